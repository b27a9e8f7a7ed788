"""The 8-bit cache's operators at limits that their own files leave out: commits of as many slots as
a call takes, and non-finite queries in requests of more than 16 rows."""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb
from jetspec_b200 import _lib

from helpers import bits_equal
from test_gpu_tree_fp8 import DEVICE, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim", [128, 64, 16])
@pytest.mark.parametrize("short", [0, 1, 7])
def test_a_commit_of_as_many_slots_as_a_call_takes(dim, short):
    n = _lib.load_library().jt_kv_fp8_commit_max_slots() - short
    blocks, block, heads = 60, 256, 2
    gen = torch.Generator(device=DEVICE).manual_seed(dim + short)
    pool, scale = jb.alloc_fp8_kv_cache(1, blocks, block, heads, dim, DEVICE)
    codes, bytes_ = pool.view(torch.uint8), scale.view(torch.uint8)
    codes.random_(0, 127, generator=gen)
    bytes_.random_(0, 255, generator=gen)
    order = torch.randperm(blocks * block, generator=gen, device=DEVICE)
    source, destination = order[:n], order[torch.randperm(n, generator=gen, device=DEVICE)]
    rows = codes.view(2, 1, -1, heads, dim).clone()
    flat = bytes_.transpose(3, 4).reshape(2, 1, -1, heads).clone()
    rows[:, :, destination] = rows[:, :, source].clone()
    flat[:, :, destination] = flat[:, :, source].clone()
    jb.copy_accepted_kv_fp8(pool, scale, source, destination, block)
    assert torch.equal(codes.view(2, 1, -1, heads, dim), rows)
    assert torch.equal(bytes_.transpose(3, 4).reshape(2, 1, -1, heads), flat)
    assert jb.read_device_errors() == 0


def test_one_slot_more_is_refused():
    n = _lib.load_library().jt_kv_fp8_commit_max_slots() + 1
    pool, scale = jb.alloc_fp8_kv_cache(1, 60, 256, 1, 16, DEVICE)
    slots = torch.arange(n, device=DEVICE)
    with pytest.raises(ValueError, match="per-call limit"):
        jb.copy_accepted_kv_fp8(pool, scale, slots, slots, 256)


@pytest.mark.parametrize("counts", [[40], [130], [33, 90]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_non_finite_queries_stay_in_their_rows(counts, dtype):
    case = Case([300] * len(counts), counts, dtype=dtype, seed=19)
    want = case.run()
    q = case.q.clone()
    q[0, 1, 5] = float("inf")
    q[7, 3, 0] = float("nan")
    q[-1, 0, 100] = float("-inf")
    case.q = q
    got = case.run()
    for at in ((0, 1), (7, 3), (-1, 0)):
        assert torch.isnan(got[at]).all()
        got[at] = want[at]
    assert bits_equal(got, want)
