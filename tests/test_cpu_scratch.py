"""Scratch of the operators that hand state from kernel to kernel: who may use which bytes when.

No GPU: the library, the stream lookup and the capture query are stood in for, and the fake
launch records the scratch that it was given and how long the call lasted.
"""
from __future__ import annotations

import threading
import time
import weakref
from types import SimpleNamespace

import pytest
import torch

from jetspec_b200 import _launch, _lib, tree_fp8, tree_gqa

KV_HEADS, GROUPS, DIM, BLOCK = 2, 4, 64, 16


class FakeLibrary:
    """Sizes by a rule like the real ones'; launches that take a while and note (start, end,
    scratch address, scratch bytes)."""

    capturing = False

    def __init__(self, seconds=0.0):
        self.seconds, self.calls = seconds, []

    def _launch(self, p, stream):
        start = time.perf_counter()
        time.sleep(self.seconds)
        p = p._obj
        self.calls.append((start, time.perf_counter(), p.workspace, p.workspace_bytes))
        return _lib.JT_OK

    jt_tree_attn_fp8_launch = jt_tree_attn_launch = _launch

    def jt_tree_attn_fp8_workspace_size(self, requests, total, heads, groups, dim):
        return 4096 + 512 * total

    def jt_tree_attn_workspace_size(self, requests, total, heads, groups, dim, out):
        out._obj.value = 4096 + 512 * total
        return _lib.JT_OK


def metadata(total):
    i32, i64 = torch.int32, torch.int64
    return SimpleNamespace(
        cu_seqlens_q=torch.tensor([0, total], dtype=i32),
        query_to_request=torch.zeros(total, dtype=i32), query_local_row=torch.arange(total).int(),
        prefix_lens=torch.zeros(1, dtype=i32), node_counts=torch.tensor([total], dtype=i32),
        block_tables=torch.zeros((1, 1), dtype=i32), tree_slots=torch.arange(total, dtype=i64),
        qq_bias=torch.zeros(total * total), qq_bias_offsets=torch.zeros(2, dtype=i64),
        block_size=BLOCK, num_requests=1, total_queries=total, node_counts_host=(total,))


def call_fp8(total):
    q = torch.zeros((total, KV_HEADS * GROUPS, DIM), dtype=torch.bfloat16)
    pool = torch.zeros((4, BLOCK, KV_HEADS, DIM), dtype=torch.uint8)
    scale = torch.zeros((4, KV_HEADS, BLOCK), dtype=torch.uint8)
    tree_fp8._launch_attention(torch.empty_like(q), q, pool, pool, scale, scale, metadata(total),
                               0.125, GROUPS)


def call_16bit(total):
    q = torch.zeros((total, KV_HEADS * GROUPS, DIM), dtype=torch.bfloat16)
    pool = torch.zeros((4, BLOCK, KV_HEADS, DIM), dtype=torch.bfloat16)
    tree_gqa.launch_tree_attention_eager(torch.empty_like(q), q, pool, pool, metadata(total),
                                         0.125, GROUPS)


@pytest.fixture
def fake(monkeypatch):
    lib = FakeLibrary()
    monkeypatch.setattr(_lib, "load_library", lambda *a: lib)
    monkeypatch.setattr(_launch, "raw_stream", lambda device: 77)
    monkeypatch.setattr(torch._C, "_cuda_isCurrentStreamCapturing", lambda: lib.capturing,
                        raising=False)
    monkeypatch.setattr(tree_fp8, "_WORKSPACE_SIZES", {})
    monkeypatch.setattr(tree_gqa, "_WORKSPACE_SIZES", {})
    return lib


@pytest.mark.parametrize("call", [call_fp8, call_16bit])
def test_threads_on_one_stream_do_not_share_scratch_at_a_time(fake, call):
    """Two calls whose launches interleave must not hold the same bytes: one's second kernel
    would read what the other's first kernel wrote."""
    fake.seconds = 0.02
    threads = [threading.Thread(target=call, args=(5,)) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    calls = sorted(fake.calls)
    assert len(calls) == 4
    for i, (_, end, address, _) in enumerate(calls):
        for start, _, other, _ in calls[i + 1:]:
            assert other != address or start >= end


@pytest.mark.parametrize("call", [call_fp8, call_16bit])
def test_a_captured_call_takes_scratch_of_its_own(fake, call, monkeypatch):
    """A graph replays whenever its owner likes: beside eager calls on the stream that it was
    captured on, and beside graphs captured there after it.  Its scratch has to come from the
    allocator at the capture (from the graph's own pool), not from what calls share."""
    made = []
    empty = torch.empty

    def counted(*args, **kwargs):
        tensor = empty(*args, **kwargs)
        if tensor.dtype == torch.uint8:
            made.append(tensor)  # kept: no address comes twice
        return tensor

    monkeypatch.setattr(torch, "empty", counted)
    call(5)
    call(5)
    fake.capturing = True
    call(5)
    call(5)
    fake.capturing = False
    call(5)
    used = [c[2] for c in fake.calls]
    assert used[0] == used[1] == used[4]
    assert len(set(used)) == 3
    assert set(used[2:4]) <= {t.data_ptr() for t in made}


@pytest.mark.parametrize("call", [call_fp8, call_16bit])
def test_scratch_stays_bounded_over_many_sizes(fake, call, monkeypatch):
    """A serving loop meets every total of packed nodes; what stays allocated after it must not
    grow with their number."""
    made = []
    empty = torch.empty

    def counted(*args, **kwargs):
        tensor = empty(*args, **kwargs)
        if tensor.dtype == torch.uint8:
            made.append((weakref.ref(tensor), tensor.numel()))
        return tensor

    monkeypatch.setattr(torch, "empty", counted)
    stream = object()  # one that no other call has used
    monkeypatch.setattr(_launch, "raw_stream", lambda device: hash(stream))
    totals = [*range(1, 200, 3), *range(200, 1, -7)]
    for total in totals:
        call(total)
    largest = max(c[3] for c in fake.calls)
    assert [c[3] for c in fake.calls] == [4096 + 512 * t for t in totals]
    held = sum(n for ref, n in made if ref() is not None)
    assert largest <= held <= 2 * largest
    assert len(made) <= 24  # allocations, not one per size


def test_remembered_sizes_stay_bounded():
    sizes = {}
    for total in range(10000):
        assert _launch.remember(sizes, (1, total), 3 * total) == 3 * total
        assert sizes[1, total] == 3 * total
    assert len(sizes) <= 4096
