"""build_request_maps against a host loop over requests and tokens: every value equal."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import jetspec_b200 as jb

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)


def host_maps(table, cached, new, free, block, max_tokens):
    """The round's maps, request by request and token by token."""
    table, width = [list(row) for row in table], len(table[0])
    slots, positions, owners, cu, taken = [], [], [], [0], 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        pages = {col: table[r][col] for col in range(min(-(-c // block), width))}
        for col in range(-(-c // block), -(-(c + n) // block)):
            page = free[taken] if taken < len(free) else -1
            taken += 1
            if col < width:
                table[r][col] = pages[col] = page
        for p in range(c, c + n):
            page = pages.get(p // block, -1)
            slots.append(page * block + p % block if page >= 0 else -1)
            positions.append(p)
            owners.append(r)
        cu.append(cu[-1] + n)
    pad = max_tokens - len(slots)
    lens = [max(c, 0) + max(n, 0) for c, n in zip(cached, new)]
    return (table, (slots + [-1] * pad)[:max_tokens], (positions + [0] * pad)[:max_tokens],
            (owners + [-1] * pad)[:max_tokens], cu, lens, [taken])


def check(cached, new, block, *, width=None, spare=3, capacity=None, seed=0, row_pad=0):
    rng = np.random.default_rng(seed)
    cached, new = [int(c) for c in cached], [int(n) for n in new]
    have = [-(-max(c, 0) // block) for c in cached]
    need = [-(-(max(c, 0) + max(n, 0)) // block) for c, n in zip(cached, new)]
    width = max(max(need), 1) + 1 if width is None else width
    order = rng.permutation(sum(need) + max(spare, 0)).tolist()
    table = [[-1] * width for _ in cached]
    for r, h in enumerate(have):
        for col in range(h):
            page = order.pop()
            if col < width:
                table[r][col] = page
    free = order if spare >= 0 else order[:len(order) + spare]
    capacity = sum(max(n, 0) for n in new) if capacity is None else capacity

    def dev(x):
        return torch.tensor(x, dtype=torch.int32, device=DEVICE)

    backing = torch.full((len(table), width + row_pad), -7, dtype=torch.int32, device=DEVICE)
    backing[:, :width] = dev(table)
    tables = backing[:, :width]
    maps = jb.build_request_maps(tables, dev(cached), dev(new), dev(free), block,
                                 max_tokens=capacity)
    assert maps.block_tables is tables
    expected = host_maps(table, cached, new, free, block, capacity)
    for got, want in zip((tables, maps.slot_mapping, maps.positions, maps.token_to_request,
                          maps.cu_seqlens, maps.context_lens, maps.pages_taken), expected):
        assert got.tolist() == want
    assert (backing[:, width:] == -7).all()
    return maps


@pytest.mark.parametrize("block", [1, 16, 100, 256])
def test_ragged_rounds(block):
    rng = np.random.default_rng(block)
    cached = rng.integers(0, 700, size=37)
    new = rng.integers(0, 300, size=37)
    new[5] = 0
    cached[6] = 0
    check(cached, new, block, seed=block, row_pad=3)


def test_decode_round_and_page_edges():
    # The cached length ends one short of a page, on it, and one past it.
    check([255, 256, 257, 0, 1, 511, 512], [1] * 7, 256)


def test_single_request_single_token():
    check([0], [1], 256)
    check([300], [0], 256, capacity=4)


def test_padding_and_truncation():
    check([10, 20], [3, 4], 16, capacity=16)
    check([10, 20], [3, 4], 16, capacity=5)
    check([10, 20], [3, 4], 16, capacity=0)


@pytest.mark.parametrize("requests", [511, 512, 513, 3000])
def test_more_requests_than_threads(requests):
    rng = np.random.default_rng(requests)
    check(rng.integers(0, 90, size=requests), rng.integers(0, 7, size=requests), 16, seed=1)


def test_a_long_prompt_beside_decodes():
    check([0] + [100] * 20 + [7], [70001] + [1] * 20 + [30000], 64)


def test_short_free_list_and_narrow_table():
    check([30, 0, 5], [40, 40, 40], 16, spare=-2)
    maps = check([30, 0, 5], [40, 40, 40], 16, width=3)
    assert (maps.slot_mapping == -1).any()


def test_negative_lengths_count_as_zero_and_are_flagged():
    jb.read_device_errors()
    check([-5, 10], [4, -3], 16)
    assert jb.read_device_errors() & 1


def test_captured_round_replays_with_new_lengths():
    table = torch.full((2, 8), -1, dtype=torch.int32, device=DEVICE)
    cached = torch.zeros(2, dtype=torch.int32, device=DEVICE)
    new = torch.tensor([3, 5], dtype=torch.int32, device=DEVICE)
    free = torch.arange(16, dtype=torch.int32, device=DEVICE)
    jb.build_request_maps(table, cached, new, free, 4, max_tokens=16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        maps = jb.build_request_maps(table, cached, new, free, 4, max_tokens=16)
    new.copy_(torch.tensor([6, 1], dtype=torch.int32))
    table.fill_(-1)
    graph.replay()
    want = host_maps([[-1] * 8] * 2, [0, 0], [6, 1], list(range(16)), 4, 16)
    assert maps.slot_mapping.tolist() == want[1] and table.tolist() == want[0]
