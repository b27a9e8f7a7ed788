"""copy_accepted_kv_fp8: a gather before a scatter, byte for byte."""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)


def cache(layers, blocks, block, heads, dim, seed=0):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    pool, scale = jb.alloc_fp8_kv_cache(layers, blocks, block, heads, dim, DEVICE)
    pool.view(torch.uint8).random_(0, 256, generator=gen)
    scale.view(torch.uint8).random_(0, 256, generator=gen)
    return pool, scale


def expected(pool, scale, src, dst, block):
    p, s = pool.view(torch.uint8).clone(), scale.view(torch.uint8).clone()
    src, dst = src.long(), dst.long()
    rows = p[:, :, src // block, src % block].clone()
    held = s[:, :, src // block, :, src % block].clone()
    p[:, :, dst // block, dst % block] = rows
    s[:, :, dst // block, :, dst % block] = held
    return p, s


@pytest.mark.parametrize("n", [1, 5, 96, 700, 2500])
@pytest.mark.parametrize("layers,heads,dim", [(3, 8, 128), (1, 1, 64), (2, 3, 16), (2, 2, 48)])
def test_commit_matches_gather_then_scatter(n, layers, heads, dim):
    block = 64
    blocks = -(-2 * n // block) + 1
    pool, scale = cache(layers, blocks, block, heads, dim, seed=n)
    order = torch.randperm(blocks * block, device=DEVICE)
    src = order[:n]
    # Half of the destinations are other tokens' sources.
    dst = torch.cat([order[n // 2:n], order[n:n + (n - (n - n // 2))]])
    want = expected(pool, scale, src, dst, block)
    paid = jb.copy_accepted_kv_fp8(pool, scale, src, dst, block)
    assert paid == n * 2 * layers * heads * (dim + 1)
    assert torch.equal(pool.view(torch.uint8), want[0])
    assert torch.equal(scale.view(torch.uint8), want[1])


def test_int32_maps_swap_and_empty():
    pool, scale = cache(2, 2, 16, 2, 64)
    src = torch.tensor([3, 20], dtype=torch.int32, device=DEVICE)
    dst = torch.tensor([20, 3], dtype=torch.int64, device=DEVICE)
    want = expected(pool, scale, src, dst, 16)
    jb.copy_accepted_kv_fp8(pool, scale, src, dst, 16)
    assert torch.equal(pool.view(torch.uint8), want[0])
    assert torch.equal(scale.view(torch.uint8), want[1])
    assert jb.copy_accepted_kv_fp8(pool, scale, src[:0], dst[:0], 16) == 0


def test_slot_limit_and_range():
    pool, scale = cache(1, 1, 16, 1, 16)
    many = torch.zeros(12048, dtype=torch.int64, device=DEVICE)
    with pytest.raises(ValueError, match="per-call limit"):
        jb.copy_accepted_kv_fp8(pool, scale, many, many, 16)
    before = pool.view(torch.uint8).clone()
    jb.read_device_errors()
    jb.copy_accepted_kv_fp8(pool, scale, torch.tensor([99, 1], device=DEVICE),
                            torch.tensor([2, -4], device=DEVICE), 16)
    assert jb.read_device_errors() & 1
    assert torch.equal(pool.view(torch.uint8), before)
