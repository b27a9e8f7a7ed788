"""qk_norm_rope / qk_norm_rope_store against the formulas in 64 bits.

Tolerances: the kernel computes in fp32 (relative error of a rotated element a few 2^-24 of
the row's largest value, bounded here by 2^-20 of it) and rounds once: half a unit in the
last place of the output type, which for a significand of p bits is at most 2^-p of the value
(bf16 8, f16 11, fp32 24 bits), or 2^-25 for the smallest f16; an e4m3 code is within 2^-4 of the value, or half the least code 2^-10 times the
scale.
"""
from __future__ import annotations

import pytest
import torch

import jetspec_b200 as jb

pytestmark = pytest.mark.gpu
DEVICE = torch.device("cuda", 0)
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
EPS = 1e-6


def inputs(rows, q_heads, kv_heads, dim, dtype, *, seed=0, fused=True, max_position=97,
           index=torch.int64, cache_dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    width = (q_heads + 2 * kv_heads) * dim
    qkv = (torch.randn((rows, width), generator=gen) * 1.7).to(dtype).to(DEVICE)
    if fused:
        q, k, v = qkv.split([q_heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    else:
        q, k, v = (t.contiguous() for t in
                   qkv.split([q_heads * dim, kv_heads * dim, kv_heads * dim], dim=1))
    q, k, v = q.unflatten(1, (q_heads, dim)), k.unflatten(1, (kv_heads, dim)), \
        v.unflatten(1, (kv_heads, dim))
    qw = (1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype).to(DEVICE)
    kw = (1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype).to(DEVICE)
    angle = torch.rand((max_position, dim // 2), generator=gen) * 6.28
    cache = torch.cat([angle.cos(), angle.sin()], -1).to(cache_dtype).to(DEVICE)
    positions = torch.randint(0, max_position, (rows,), generator=gen).to(index).to(DEVICE)
    return q, k, v, qw, kw, positions, cache


def formula(x, weight, positions, cache):
    x, w = x.double(), weight.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w
    cos, sin = cache.double().view(cache.shape[0], -1)[positions.long()][:, None].chunk(2, -1)
    a, b = y.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def assert_rounded(got, want, dtype):
    assert got.dtype == dtype and got.shape == want.shape
    least = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bound = ROUND[dtype] * want.abs() + 2.0 ** -20 * want.abs().amax(-1, keepdim=True) + least
    assert ((got.double() - want).abs() <= bound).all()


def assert_quantized(codes, scale, want):
    """codes [n, h, d], scale [n, h] against rows ``want``: the least sufficient power of two,
    and codes within half a spacing."""
    s, amax = scale.double(), want.abs().amax(-1)
    slack = 1 + 2.0 ** -20
    assert (amax <= 448 * s * slack).all()
    assert ((amax == 0) | (amax * slack > 224 * s)).all()
    assert torch.equal(torch.exp2(torch.round(torch.log2(s))), s)
    held = codes.double() * s[..., None]
    bound = torch.maximum(want.abs() * 2.0 ** -4, 2.0 ** -10 * s[..., None]) \
        + 2.0 ** -20 * amax[..., None]
    assert ((held - want).abs() <= bound).all()


SHAPES = [(1, 4, 1, 128), (7, 32, 8, 128), (129, 14, 2, 64), (33, 3, 3, 256), (5, 6, 2, 96),
          (9, 2, 1, 2), (4, 5, 5, 500), (2500, 8, 2, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,q_heads,kv_heads,dim", SHAPES)
def test_norm_and_rotation(rows, q_heads, kv_heads, dim, dtype):
    q, k, _, qw, kw, positions, cache = inputs(rows, q_heads, kv_heads, dim, dtype, seed=dim)
    got_q, got_k = jb.qk_norm_rope(q, k, qw, kw, positions, cache, EPS)
    assert_rounded(got_q, formula(q, qw, positions, cache), dtype)
    assert_rounded(got_k, formula(k, kw, positions, cache), dtype)


def pools(rows, kv_heads, dim, dtype, block, seed=3):
    gen = torch.Generator().manual_seed(seed)
    blocks = -(-rows // block) + 2
    slots = torch.randperm(blocks * block, generator=gen)[:rows].to(DEVICE)
    if rows > 2:
        slots[1] = -1
    if dtype is None:
        pool, scale = jb.alloc_fp8_kv_cache(1, blocks, block, kv_heads, dim, DEVICE)
        return slots, pool[0, 0], pool[1, 0], scale[0, 0], scale[1, 0]
    pool = torch.full((2, blocks, block, kv_heads, dim), 5.0, dtype=dtype, device=DEVICE)
    return slots, pool[0], pool[1], None, None


def gather(pool, slots, block):
    return pool.view(torch.uint8 if pool.dtype.itemsize == 1 else pool.dtype)[
        slots // block, slots % block].view(pool.dtype)


def gather_scale(scale, slots, block):
    return scale.view(torch.uint8)[slots // block, :, slots % block].view(scale.dtype)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("block", [16, 256])
@pytest.mark.parametrize("rows,q_heads,kv_heads,dim", SHAPES)
def test_store_8bit(rows, q_heads, kv_heads, dim, block, index):
    q, k, v, qw, kw, positions, cache = inputs(rows, q_heads, kv_heads, dim, torch.bfloat16,
                                               seed=rows, index=index)
    slots, kp, vp, ks, vs = pools(rows, kv_heads, dim, None, block)
    out = jb.qk_norm_rope_store(q, k, v, qw, kw, positions, cache, kp, vp, slots.to(index), EPS,
                                k_scale=ks, v_scale=vs)
    assert_rounded(out, formula(q, qw, positions, cache), torch.bfloat16)
    live = slots >= 0
    at = slots[live]
    assert_quantized(gather(kp, at, block), gather_scale(ks, at, block),
                     formula(k, kw, positions, cache)[live])
    assert_quantized(gather(vp, at, block), gather_scale(vs, at, block), v[live].double())
    # Nothing else was written: every other slot still holds zeros with scale one.
    untouched = torch.ones(kp.shape[0] * block, dtype=torch.bool, device=DEVICE)
    untouched[at] = False
    for pool, scale in ((kp, ks), (vp, vs)):
        assert (pool.view(torch.uint8).flatten(0, 1)[untouched] == 0).all()
        assert (scale.view(torch.uint8).transpose(1, 2).flatten(0, 1)[untouched] == 127).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,q_heads,kv_heads,dim", SHAPES[:6])
def test_store_operand_type(rows, q_heads, kv_heads, dim, dtype):
    q, k, v, qw, kw, positions, cache = inputs(rows, q_heads, kv_heads, dim, dtype, seed=rows + 1)
    slots, kp, vp, _, _ = pools(rows, kv_heads, dim, dtype, 16)
    out = jb.qk_norm_rope_store(q, k, v, qw, kw, positions, cache, kp, vp, slots, EPS)
    assert_rounded(out, formula(q, qw, positions, cache), dtype)
    live = slots >= 0
    at = slots[live]
    assert_rounded(gather(kp, at, 16), formula(k, kw, positions, cache)[live], dtype)
    assert torch.equal(gather(vp, at, 16), v[live])
    untouched = torch.ones(kp.shape[0] * 16, dtype=torch.bool, device=DEVICE)
    untouched[at] = False
    assert (kp.flatten(0, 1)[untouched] == 5).all() and (vp.flatten(0, 1)[untouched] == 5).all()


def test_exponent_edges():
    """Rows whose largest value sits on, just under and just over 448 * 2^e, rows of zeros,
    the smallest and the largest finite values: V rows are quantised as they come."""
    dim, dtype = 128, torch.float32
    big = torch.finfo(dtype).max
    tops = [448.0, 448.0 * (1 + 2 ** -22), 448.0 * (1 - 2 ** -22), 1.0, 1.75, 1.7500001, 0.0,
            1e-30, 2.0 ** -149, 2.0 ** -126, big, -448.0, 3.5e-38]
    v = torch.zeros((len(tops), 1, dim), dtype=dtype)
    v[:, 0, 77] = torch.tensor(tops)
    v[:, 0, 3] = torch.tensor(tops) / 7
    v = v.to(DEVICE)
    q, k, _, qw, kw, positions, cache = inputs(len(tops), 1, 1, dim, dtype)
    _, kp, vp, ks, vs = pools(len(tops), 1, dim, None, 16)
    slots = torch.arange(len(tops), device=DEVICE)
    jb.qk_norm_rope_store(q, k, v, qw, kw, positions, cache, kp, vp, slots, EPS, k_scale=ks,
                          v_scale=vs)
    byte = vs.view(torch.uint8)[0, 0, :len(tops)].long()
    for i, top in enumerate(tops):
        e = int(byte[i]) - 127
        a = abs(float(v[i, 0, 77]))
        if a == 0.0:
            assert e == 0
        elif a >= 2.0 ** -118:
            assert a <= 448 * 2.0 ** e and a > 224 * 2.0 ** e, top
        else:
            assert e >= -127 and a <= 448 * 2.0 ** e
    held = vp.view(torch.uint8)[0, :len(tops)].view(vp.dtype).double() \
        * torch.exp2((byte - 127).double())[:, None, None]
    bound = torch.maximum(v.double().abs() * 2.0 ** -4,
                          torch.exp2((byte - 127).double() - 10)[:, None, None])
    assert ((held - v.double()).abs() <= bound).all()


def test_non_finite_rows_read_back_as_nan():
    q, k, v, qw, kw, positions, cache = inputs(4, 2, 2, 128, torch.bfloat16, fused=False)
    v[1, 0, 5] = float("inf")
    k[2, 1, 9] = float("nan")
    slots, kp, vp, ks, vs = pools(4, 2, 128, None, 16)
    slots = torch.arange(4, device=DEVICE)
    out = jb.qk_norm_rope_store(q, k, v, qw, kw, positions, cache, kp, vp, slots, EPS,
                                k_scale=ks, v_scale=vs)
    assert torch.isfinite(out).all()
    kk = gather_scale(ks, slots, 16).float()
    vv = gather_scale(vs, slots, 16).float()
    assert torch.isnan(kk).nonzero().tolist() == [[2, 1]]
    assert torch.isnan(vv).nonzero().tolist() == [[1, 0]]
    assert (gather(vp, slots, 16).view(torch.uint8)[1, 0] == 0).all()
    assert torch.isnan(jb.dequantize_kv(vp, vs)[0, 1, 0]).all()


def test_zero_rows_and_in_place():
    q, k, v, qw, kw, positions, cache = inputs(6, 4, 2, 128, torch.bfloat16)
    empty = jb.qk_norm_rope(q[:0], k[:0], qw, kw, positions[:0], cache, EPS)
    assert empty[0].shape == (0, 4, 128) and empty[1].shape == (0, 2, 128)
    want = jb.qk_norm_rope(q, k, qw, kw, positions, cache, EPS)
    got = jb.qk_norm_rope(q, k, qw, kw, positions, cache, EPS, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    # A head of zeros stays zero (eps keeps the norm finite).
    z = torch.zeros_like(want[0])
    assert (jb.qk_norm_rope(z, want[1], qw, kw, positions, cache, EPS)[0] == 0).all()


def test_unaligned_views_and_other_cache_types():
    q, k, v, qw, kw, positions, cache = inputs(11, 4, 2, 128, torch.bfloat16)
    wide = torch.randn((11, 4, 131), device=DEVICE).bfloat16()
    odd = wide[..., 1:129]  # rows start on odd elements
    got, _ = jb.qk_norm_rope(odd, k, qw, kw, positions, cache, EPS)
    assert_rounded(got, formula(odd, qw, positions, cache), torch.bfloat16)
    half = cache.bfloat16().view(-1, 1, 128)
    got, _ = jb.qk_norm_rope(q, k, qw.float(), kw.float(), positions, half, EPS)
    assert_rounded(got, formula(q, qw, positions, half), torch.bfloat16)


def test_out_of_range_slots_and_positions_are_flagged():
    q, k, v, qw, kw, positions, cache = inputs(3, 2, 1, 128, torch.bfloat16)
    slots, kp, vp, ks, vs = pools(3, 1, 128, None, 16)
    slots = torch.tensor([0, 10 ** 6, 2 ** 40], device=DEVICE)
    jb.read_device_errors()
    jb.qk_norm_rope_store(q, k, v, qw, kw, positions, cache, kp, vp, slots, EPS, k_scale=ks,
                          v_scale=vs)
    assert jb.read_device_errors() & 1
    assert (vp.view(torch.uint8)[0, 1:] == 0).all()
    jb.qk_norm_rope(q, k, qw, kw, positions + 1000, cache, EPS)
    assert jb.read_device_errors() & 1


def test_another_stream():
    q, k, v, qw, kw, positions, cache = inputs(64, 8, 2, 128, torch.bfloat16)
    want = jb.qk_norm_rope(q, k, qw, kw, positions, cache, EPS)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = jb.qk_norm_rope(q, k, qw, kw, positions, cache, EPS)
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
