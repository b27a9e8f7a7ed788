"""Requests that packed_tree_attention_fp8 does not take: their rows are zeros and a device error bit
is set, whatever the output's memory held; the other requests' rows are what they are alone.
"""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb
from jetspec_b200 import tree_fp8

from helpers import bits_equal
from test_gpu_tree_fp8 import DEVICE, Case
from test_gpu_tree_fp8_few import namespace

pytestmark = pytest.mark.gpu


def run(case, meta, dtype=torch.bfloat16):
    """The launch into memory that holds sevens, with sevens before and after it."""
    shape = (case.q.shape[0] + 16, *case.q.shape[1:])
    memory = torch.full(shape, 7.0, dtype=dtype, device=DEVICE)
    out = memory[8:-8]
    tree_fp8._launch_attention(out, case.q, case.k, case.v, case.ks, case.vs, meta, case.scale,
                               case.batch.groups)
    torch.cuda.synchronize()
    assert (memory[:8] == 7).all() and (memory[-8:] == 7).all()
    return out


def rows(case, r):
    o = case.meta.cu_seqlens_q.tolist()
    return slice(o[r], o[r + 1])


@pytest.mark.parametrize("counts", [[3, 1030, 40], [1100], [64, 1025, 2000, 1]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_trees_of_more_than_1024_nodes(counts, dtype):
    """Known too large on the device only: the host's counts are not given."""
    case = Case([200 + i for i in range(len(counts))], counts, kv_heads=1, groups=2, seed=31)
    meta = namespace(case.meta, node_counts_host=None)
    jb.read_device_errors()
    got = run(case, meta, dtype)
    assert jb.read_device_errors() == 2
    small = [r for r, n in enumerate(counts) if n <= 1024]
    for r, n in enumerate(counts):
        if n > 1024:
            assert (got[rows(case, r)] == 0).all()
    if small:
        case.run = lambda **kw: got
        case.check(small)


@pytest.mark.parametrize("groups,counts,known", [(1, (5, 9, 4), True), (4, (5, 9, 4), False),
                                                 (4, (50, 90, 40), True), (4, (50, 3, 1), False)])
def test_nodes_past_the_packed_rows(groups, counts, known):
    """Device counts and offsets that leave the rows of the call: nothing is written past them."""
    case = Case([300, 40, 900], counts, kv_heads=2, groups=groups, seed=32)
    total, m = sum(counts), case.meta
    late = total - counts[2] + 3  # the last request begins three rows on
    bias = torch.cat([m.qq_bias.view(-1), m.qq_bias.new_zeros(4096)])
    for cu, bad in (([0, counts[0], late, total], [2]), ([-2, counts[0], total - counts[2], total], [0]),
                    ([0, counts[0], total, total], [2])):
        meta = namespace(m, cu_seqlens_q=torch.tensor(cu, dtype=torch.int32, device=DEVICE),
                         qq_bias=bias, **({} if known else {"node_counts_host": None}))
        jb.read_device_errors()
        got = run(case, meta)
        assert jb.read_device_errors() == 1
        good = [r for r in range(3) if r not in bad]
        for r in bad:
            lo, hi = max(cu[r], 0), min(cu[r] + counts[r], total)
            assert (got[lo:hi] == 0).all()
        case.run = lambda **kw: got
        case.check(good)
    counts_up = m.node_counts.clone()
    counts_up[2] += 6
    meta = namespace(m, node_counts=counts_up, qq_bias=bias,
                     **({} if known else {"node_counts_host": None}))
    got = run(case, meta)
    assert jb.read_device_errors() == 1
    assert (got[rows(case, 2)] == 0).all()
    case.run = lambda **kw: got
    case.check([0, 1])


@pytest.mark.parametrize("groups,host,device,taken", [
    (4, (4, 4, 3), (1, 9, 1), (0, 2)),          # only few rows known: a tree of 36 is not taken
    (4, (2, 2, 1), (1, 3, 1), (0, 2)),          # up to 8 rows known: nor is one of 12
    (4, (40, 20, 30), (44, 3, 43), (0, 2)),     # only large trees known: nor one of 12
    (4, (40, 20, 30), (20, 30, 40), (0, 1, 2)),  # other counts that the same kernel takes
    (4, (3, 40, 5), (40, 3, 5), (0, 1, 2)),     # both kernels run: all are taken
])
def test_host_counts_that_are_not_the_devices(groups, host, device, taken):
    case = Case([300, 40, 900], device, kv_heads=2, groups=groups, seed=33)
    assert sum(host) == sum(device)
    meta = namespace(case.meta, node_counts_host=host)
    jb.read_device_errors()
    got = run(case, meta)
    assert jb.read_device_errors() == (0 if len(taken) == 3 else 1)
    for r in range(3):
        if r not in taken:
            assert (got[rows(case, r)] == 0).all()
    case.run = lambda **kw: got
    case.check(list(taken))


def test_a_tree_above_1024_nodes_where_few_rows_are_known():
    case = Case([300, 40], [1030, 2], kv_heads=2, groups=1, seed=34)
    jb.read_device_errors()
    got = run(case, namespace(case.meta, node_counts_host=(8, 2)))
    assert jb.read_device_errors() == 2
    assert (got[:1030] == 0).all()
    case.run = lambda **kw: got
    case.check([1])


@pytest.mark.parametrize("groups,counts", [(1, (5, 9, 4)), (4, (50, 3, 40))])
@pytest.mark.parametrize("known", [True, False])
@pytest.mark.parametrize("bad", [0, 2])
def test_counts_that_the_bias_does_not_hold(groups, counts, known, bad):
    """Offsets that give a request a smaller matrix than its nodes': it is refused, not read past."""
    case = Case([300, 40, 900], counts, kv_heads=2, groups=groups, seed=35)
    offsets = case.meta.qq_bias_offsets.clone()
    if bad == 0:
        offsets[0] += 1
    else:
        offsets[3] -= 1
    meta = namespace(case.meta, qq_bias_offsets=offsets,
                     **({} if known else {"node_counts_host": None}))
    jb.read_device_errors()
    got = run(case, meta)
    assert jb.read_device_errors() == 1
    assert (got[rows(case, bad)] == 0).all()
    case.run = lambda **kw: got
    case.check([r for r in range(3) if r != bad])
