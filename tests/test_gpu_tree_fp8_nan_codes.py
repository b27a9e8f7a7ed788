"""e4m3's NaN codes (0x7f, 0xff) in the 8-bit cache read as NaN, as dequantize_kv reads them, for the
rows that see their key, and reach no other row, in requests of few rows and of many alike.

A NaN code of K makes the whole row NaN, one of V its element; in the 128-key tile in which the
prefix ends and the tree begins (and in the tiles after it) one of V makes the whole row NaN too.
"""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb

from helpers import bits_equal
from test_gpu_tree_fp8 import Case

pytestmark = pytest.mark.gpu

PREFIX, DIM_AT = 700, 37
SIZES = [([2], 4), ([16], 1), ([1], 16), ([40], 4), ([130], 4)]


@pytest.mark.parametrize("counts,groups", SIZES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("block", [256, 16, 100])
@pytest.mark.parametrize("pool,code", [("k", 0x7F), ("k", 0xFF), ("v", 0x7F), ("v", 0xFF)])
def test_in_the_prefix(counts, groups, dtype, block, pool, code):
    """At keys of unmasked tiles (the first, one of the middle, the last) and of the tile in which
    the prefix ends."""
    case = Case([PREFIX], counts, groups=groups, dtype=dtype, block=block, seed=21)
    want = case.run()
    codes = getattr(case, pool).view(torch.uint8)
    for position in (0, 300, 639, 640, PREFIX - 1):
        slot = (case.batch.block_tables[0][position // block], position % block, 0, DIM_AT)
        kept = codes[slot].clone()
        codes[slot] = code
        got = case.run()
        codes[slot] = kept
        nan = torch.isnan(got)
        assert nan[:, :groups, DIM_AT].all()
        if pool == "k" or position >= 640:
            assert nan[:, :groups].all()
        else:
            nan[:, :groups, DIM_AT] = False
            assert not nan.any()
            got[:, :groups, DIM_AT] = want[:, :groups, DIM_AT]
            assert bits_equal(got, want)
        assert bits_equal(got[:, groups:], want[:, groups:])
    assert bits_equal(case.run(), want)
    assert jb.read_device_errors() == 0


@pytest.mark.parametrize("counts,groups", [([16], 1), ([40], 4), ([130], 4)])
@pytest.mark.parametrize("pool", ["k", "v"])
def test_in_the_tree(counts, groups, pool):
    case = Case([PREFIX], counts, groups=groups, seed=22)
    want = case.run()
    block, n = case.batch.block_size, counts[0]
    seen = case.meta.qq_bias.view(n, n) == 0
    for node in (0, 3, n - 1):
        slot = int(case.meta.tree_slots[node])
        codes = getattr(case, pool).view(torch.uint8)
        at = (slot // block, slot % block, 1, DIM_AT)
        kept = codes[at].clone()
        codes[at] = 0x7F
        got = case.run()
        codes[at] = kept
        rows = seen[:, node].clone()
        rows[:node] = False
        assert rows.any() and torch.isnan(got[rows][:, groups:]).all()
        assert bits_equal(got[~rows], want[~rows])
        assert bits_equal(got[:, :groups], want[:, :groups])


@pytest.mark.parametrize("counts", [[1], [4], [40], [130], [2, 70]])
@pytest.mark.parametrize("out", [None, torch.float32])
def test_in_requests_cut_between_multiprocessors(counts, out):
    case = Case([30011] * len(counts), counts, kv_heads=3, seed=23)
    want = case.run(output_dtype=out)
    block, groups, n = case.batch.block_size, case.batch.groups, counts[0]
    codes = case.v.view(torch.uint8)
    for position, node in ((10, None), (15000, None), (30010, None), (None, n - 1)):
        if node is None:
            at = (case.batch.block_tables[0][position // block], position % block, 2, DIM_AT)
        else:
            slot = int(case.meta.tree_slots[node])
            at = (slot // block, slot % block, 2, DIM_AT)
        kept = codes[at].clone()
        codes[at] = 0xFF
        got = case.run(output_dtype=out)
        codes[at] = kept
        hit = torch.zeros_like(got, dtype=torch.bool)
        rows = slice(0, n) if node is None else slice(n - 1, n)  # the last node: its own row alone
        dims = DIM_AT if position in (10, 15000) else slice(None)
        hit[rows, 2 * groups:, dims] = True
        assert torch.equal(torch.isnan(got), hit)
        assert torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("counts", [[2], [40]])
def test_beside_a_key_without_a_place(counts):
    """In a tile of which another page is missing."""
    case = Case([PREFIX], counts, block=16, seed=24)
    case.meta.block_tables[0, 3] = -1
    want = case.run()
    codes = case.v.view(torch.uint8)
    codes[case.batch.block_tables[0][4], 2, 0, DIM_AT] = 0x7F
    got = case.run()
    hit = torch.zeros_like(got, dtype=torch.bool)
    hit[:, :case.batch.groups, DIM_AT] = True
    assert torch.equal(torch.isnan(got), hit)
    assert torch.equal(got[~hit], want[~hit])
    assert jb.read_device_errors() == 1
