"""packed_tree_attention_fp8 against softmax attention in 64 bits over the dequantised cache.

Tolerance, element by element, with w the exact weights, A = sum w |v| and out = sum w v:

* queries enter as sums of e4m3 terms, off by at most 2^-18 of the row's largest |q|, and the
  products accumulate in fp32: a score is off by at most d = scale * 2^-17 * max|q| * sum|k|
  (largest over the keys seen), a weight by a factor 1 +- 2 d;
* BF16 queries and output: weights rounded to bf16 (2^-8) and exp2 within 2^-13: the sum is
  off by (2^-8 + 2^-12 + 2 d) A, and its rounding adds 2^-8 |out|;
* FP16 or FP32 output: weights kept to 16 bits, exp2 within 2^-20: (2^-13 + 2 d) A, and
  2^-11 |out| for the FP16 rounding (2^-25 at its smallest).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import jetspec_b200 as jb
from jetspec_b200 import workloads

from helpers import bits_equal

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)


def quantize(x):
    """e4m3 codes and scale bytes of fp32 rows, by the definition."""
    amax = x.abs().amax(-1)
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, 448.0) / 448.0)).clamp(-127, 127)
    codes = (x * torch.exp2(-e.double())[..., None]).float().clamp(-448, 448)
    return codes.to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


class Case:
    """A batch over an 8-bit cache whose unowned slots hold NaN codes and NaN scales."""

    def __init__(self, prefixes, counts, *, kv_heads=2, groups=4, dim=128, block=256, seed=5,
                 dtype=torch.bfloat16, v_std=1.0, q_std=1.0, num_blocks=None):
        rng = np.random.default_rng(seed)
        parents = [workloads.random_parents(rng, int(c), 8) for c in counts]
        self.batch = workloads.build_batch(prefixes, parents, block_size=block,
                                           num_kv_heads=kv_heads, groups=groups, head_dim=dim,
                                           seed=seed, num_blocks=num_blocks)
        b = self.batch
        gen = torch.Generator(device=DEVICE).manual_seed(seed)
        live = torch.from_numpy(b.live_slots()).to(DEVICE)
        # One layer out of a cache of two: pools and scales are strided views.
        pool, scale = jb.alloc_fp8_kv_cache(2, b.num_blocks, block, kv_heads, dim, DEVICE)
        self.cache = pool, scale
        pool.view(torch.uint8)[:, 1].fill_(255)
        scale.view(torch.uint8)[:, 1].fill_(255)
        for axis, std in ((0, 1.0), (1, v_std)):
            rows = torch.randn((live.numel(), kv_heads, dim), generator=gen, device=DEVICE) * std
            rows *= torch.exp(0.7 * torch.randn(rows.shape[:2], generator=gen, device=DEVICE))[..., None]
            codes, byte = quantize(rows)
            pool.view(torch.uint8)[axis, 1, live // block, live % block] = codes.view(torch.uint8)
            scale.view(torch.uint8)[axis, 1, live // block, :, live % block] = byte
        self.k, self.v, self.ks, self.vs = pool[0, 1], pool[1, 1], scale[0, 1], scale[1, 1]
        q_heads = kv_heads * groups
        fused = torch.randn((b.total_queries, (q_heads + 3) * dim), generator=gen, device=DEVICE)
        self.q = (fused * q_std).to(dtype)[:, :q_heads * dim].unflatten(1, (q_heads, dim))
        self.meta = b.metadata(DEVICE)
        self.scale = dim ** -0.5

    def run(self, **kwargs):
        return jb.packed_tree_attention_fp8(self.q, self.k, self.v, self.ks, self.vs, self.meta,
                                            self.scale, self.batch.groups, **kwargs)

    def rows(self, pool, scale, slots):
        block = self.batch.block_size
        codes = pool.view(torch.uint8)[slots // block, slots % block].view(pool.dtype).double()
        byte = scale.view(torch.uint8)[slots // block, :, slots % block].double()
        factor = torch.where(byte == 255, torch.nan, torch.exp2(byte - 127))
        return codes * factor[..., None]

    def exact(self, requests=None):
        """(out, bound on the weighted sum's error but for its rounding, d) in 64 bits."""
        b, m = self.batch, self.meta
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=DEVICE)
        spread, shift = torch.zeros_like(out), torch.zeros_like(out[..., :1])
        offsets, biases = m.cu_seqlens_q.tolist(), m.qq_bias_offsets.tolist()
        for r in range(b.num_requests) if requests is None else requests:
            lo, hi, p = offsets[r], offsets[r + 1], b.prefix_lens[r]
            t = hi - lo
            pos = torch.arange(p, device=DEVICE)
            table = torch.tensor(b.block_tables[r] or [0], device=DEVICE)
            slots = torch.cat([table[pos // b.block_size] * b.block_size + pos % b.block_size,
                               m.tree_slots[lo:hi]])
            k, v = self.rows(self.k, self.ks, slots), self.rows(self.v, self.vs, slots)
            seen = torch.ones((t, p + t), dtype=torch.bool, device=DEVICE)
            seen[:, p:] = (m.qq_bias[biases[r]:biases[r + 1]].view(t, t) == 0).tril()
            q = self.q[lo:hi].double().unflatten(1, (-1, b.groups))
            for h in range(k.shape[1]):
                s = torch.einsum("tgd,kd->tgk", q[:, h], k[:, h]) * self.scale
                s = torch.where(seen[:, None], s, -torch.inf)
                top = s.amax(-1, keepdim=True)
                w = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
                w = torch.where(seen[:, None], w, 0.0)
                w = w / torch.where(w.sum(-1, keepdim=True) == 0, 1.0, w.sum(-1, keepdim=True))
                # A key that is not seen contributes nothing, whatever its row holds.
                vv = torch.where(seen[:, None, :, None], v[:, h], 0.0)
                rows = slice(h * b.groups, (h + 1) * b.groups)
                out[lo:hi, rows] = (w[..., None] * vv).sum(2)
                spread[lo:hi, rows] = (w[..., None] * vv.abs()).sum(2)
                kk = torch.where(seen[:, None], k[:, h].abs().sum(-1), 0.0).amax(-1)
                shift[lo:hi, rows] = (self.scale * 2.0 ** -17 * q[:, h].abs().amax(-1)
                                      * kk)[..., None]
        return out, spread, shift

    def check(self, requests=None, **kwargs):
        got = self.run(**kwargs)
        out, spread, shift = self.exact(requests)
        wide = got.dtype != torch.bfloat16
        bound = ((2.0 ** -13 if wide else 2.0 ** -8 + 2.0 ** -12) + 2 * shift) * spread
        if got.dtype != torch.float32:
            bound = bound + (2.0 ** -11 if wide else 2.0 ** -8) * out.abs() + 2.0 ** -25
        if requests is not None:
            o = self.meta.cu_seqlens_q.tolist()
            rows = torch.cat([torch.arange(o[r], o[r + 1], device=DEVICE) for r in requests])
            got, out, bound = got[rows], out[rows], bound[rows]
        nan = torch.isnan(out)
        assert torch.equal(torch.isnan(got), nan)
        diff = (got.double() - out).abs()
        assert (nan | (diff <= bound)).all(), \
            f"largest error over bound {(diff / bound)[~nan].max().item():.3f}"
        assert jb.read_device_errors() == 0
        return got


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 127, 128, 129, 255, 256, 257, 640, 2048])
def test_prefix_lengths_at_tile_and_page_edges(prefix):
    Case([prefix, 300, prefix + 1], [17, 1, 64], seed=prefix).check()


@pytest.mark.parametrize("counts", [[1], [1, 1, 1, 1, 1], [2, 31, 32, 33], [63, 64, 65],
                                    [127, 128, 129, 1], [200, 7], [500], [1024]])
def test_node_counts(counts):
    Case([37 * i + 5 for i in range(len(counts))], counts, seed=len(counts), kv_heads=1).check()


@pytest.mark.parametrize("kv_heads,groups", [(1, 1), (8, 4), (2, 7), (3, 5), (1, 16), (1, 128),
                                             (2, 3), (5, 1), (1, 100)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_head_layouts(kv_heads, groups, dtype):
    Case([200, 0, 513], [9, 33, 1], kv_heads=kv_heads, groups=groups, dtype=dtype,
         seed=groups).check()


@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_head_dims(dim):
    Case([300, 64], [40, 3], dim=dim, seed=dim).check()


@pytest.mark.parametrize("block", [1, 7, 16, 32, 64, 100, 128, 256, 512])
def test_page_sizes(block):
    Case([333, 64, 0], [20, 70, 5], block=block, seed=block).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("out", [None, torch.float32])
def test_types(dtype, out):
    case = Case([1000, 129], [64, 10], dtype=dtype, seed=11)
    assert case.check(output_dtype=out).dtype == (out or dtype)


@pytest.mark.parametrize("counts", [[1], [4], [64], [130]])
def test_one_long_request(counts):
    Case([30011], counts, kv_heads=2, seed=23).check()


def test_many_ragged_requests():
    rng = np.random.default_rng(7)
    prefixes = np.exp(rng.uniform(0, np.log(3000), size=150)).astype(int).tolist()
    counts = rng.choice([1, 2, 5, 16, 40, 64, 90], size=150).tolist()
    Case(prefixes, counts, kv_heads=2, seed=7).check()


def test_decode_batch():
    rng = np.random.default_rng(8)
    Case(rng.integers(1, 5000, size=40).tolist(), [1] * 40, kv_heads=8, seed=8).check()


def test_large_and_small_magnitudes():
    # Peaked rows, and values whose scales lie far from one.
    Case([700], [40], q_std=20.0, v_std=1e-20, seed=3).check()
    Case([700], [40], q_std=1e-3, v_std=1e20, seed=4).check(output_dtype=torch.float32)


def test_off_branch_rows_never_arrive():
    """NaN, and finite values near the top of the range, in nodes a row does not see."""
    case = Case([130], [30], seed=9)
    want = case.check()
    block = case.batch.block_size
    seen = case.meta.qq_bias.view(30, 30) == 0
    for node, byte in ((7, 255), (12, 254)):
        slot = int(case.meta.tree_slots[node])
        for scale in (case.ks, case.vs):
            scale.view(torch.uint8)[slot // block, :, slot % block] = byte
    case.k.view(torch.uint8)[int(case.meta.tree_slots[7]) // block,
                             int(case.meta.tree_slots[7]) % block] = 0x7F
    got = case.run()
    apart = ~(seen[:, 7] | seen[:, 12])
    assert apart.any()
    assert bits_equal(got[apart], want[apart])
    assert torch.isnan(got[seen[:, 7]]).all()


def test_a_nan_row_in_the_prefix_reaches_every_row():
    case = Case([300, 200], [5, 5], seed=10)
    page = case.batch.block_tables[0][1]
    case.vs.view(torch.uint8)[page, 0, 3] = 255
    got = case.check()
    groups = case.batch.groups
    assert torch.isnan(got[:5, :groups]).all()
    assert torch.isfinite(got[:5, groups:]).all() and torch.isfinite(got[5:]).all()


def test_rows_that_see_nothing_give_zeros():
    case = Case([0, 0], [12, 3], seed=12)
    case.meta.qq_bias.view(-1)[:144].view(12, 12)[4] = -torch.inf
    got = case.check()
    assert (got[4] == 0).all() and (got[5] != 0).any()


def test_a_request_without_nodes():
    case = Case([100, 50, 80], [6, 9, 4], seed=13)
    want = case.run()
    m = case.meta
    from types import SimpleNamespace

    def with_empty(x, at, value):
        return torch.cat([x[:at], x.new_tensor([value]), x[at:]])

    width = m.block_tables.shape[1]
    meta = SimpleNamespace(
        cu_seqlens_q=with_empty(m.cu_seqlens_q, 1, 6), node_counts=with_empty(m.node_counts, 1, 0),
        query_to_request=torch.where(m.query_to_request >= 1, m.query_to_request + 1,
                                     m.query_to_request).int(),
        query_local_row=m.query_local_row, prefix_lens=with_empty(m.prefix_lens, 1, 70),
        block_tables=torch.cat([m.block_tables[:1], m.block_tables.new_full((1, width), -1),
                                m.block_tables[1:]]),
        tree_slots=m.tree_slots, qq_bias=m.qq_bias,
        qq_bias_offsets=with_empty(m.qq_bias_offsets, 1, 36), block_size=m.block_size,
        total_queries=m.total_queries, num_requests=4, node_counts_host=(6, 0, 9, 4))
    got = jb.packed_tree_attention_fp8(case.q, case.k, case.v, case.ks, case.vs, meta, case.scale,
                                       case.batch.groups)
    assert torch.allclose(got.float(), want.float(), rtol=2.0 ** -6, atol=1e-6)
    assert jb.read_device_errors() == 0


def test_offsets_past_32_bits():
    """A pool of more than 4 GiB: the request's pages lie at both ends."""
    case = Case([2000], [20], kv_heads=8, seed=14, num_blocks=17000)
    assert case.k.stride(0) * case.k.shape[0] > 1 << 32
    case.check()


def test_repeats_are_identical_and_streams_are_respected():
    case = Case([9000, 300, 20], [64, 3, 128], seed=15)
    want = case.run()
    for _ in range(3):
        assert bits_equal(case.run(), want)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = case.run()
    torch.cuda.current_stream().wait_stream(stream)
    assert bits_equal(got, want)


def test_captured_call_replays_with_new_lengths():
    case = Case([700, 300], [20, 33], seed=16)
    case.run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = case.run()
    graph.replay()
    assert bits_equal(out, case.run())
    case.meta.prefix_lens.copy_(torch.tensor([65, 290], dtype=torch.int32))
    graph.replay()
    case.batch.prefix_lens[:] = [65, 290]
    assert bits_equal(out, case.check())


def test_index_errors_are_flagged_and_skipped():
    case = Case([300], [5], seed=17)
    jb.read_device_errors()
    case.meta.block_tables[0, 1] = 10 ** 6
    case.run()
    assert jb.read_device_errors() & 1


def test_refusals():
    case = Case([10], [3], seed=18)
    m, s, g = case.meta, case.scale, case.batch.groups

    def call(q=case.q, k=case.k, v=case.v, ks=case.ks, vs=case.vs, scale=s, groups=g, **kw):
        return jb.packed_tree_attention_fp8(q, k, v, ks, vs, m, scale, groups, **kw)

    for match, kw in [("metadata", dict(q=case.q[:2])), ("geometry", dict(v=case.v[:1])),
                      ("e4m3", dict(k=case.k.view(torch.uint8))),
                      ("e8m0", dict(ks=case.ks.view(torch.uint8))),
                      ("kv_heads", dict(vs=case.vs[:, :1], ks=case.ks[:, :1])),
                      ("grouping", dict(groups=3)), ("BF16 or FP16", dict(q=case.q.float())),
                      ("output dtype", dict(output_dtype=torch.float16)),
                      ("scale must be positive", dict(scale=0.0)),
                      ("scale must be positive", dict(scale=float("nan"))),
                      ("head dim", dict(q=case.q[..., :64])),
                      ("CUDA", dict(q=case.q.cpu()))]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
