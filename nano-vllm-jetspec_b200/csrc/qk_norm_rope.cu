// RMS norm of every query and key head with the position rotation in the same pass, and
// (optionally) the K / V rows written into the paged cache, plain or 8-bit.
//
//   y = x * rsqrt(mean(x^2) + eps) * w                      over one head's D elements
//   out = [y1 * cos - y2 * sin, y2 * cos + y1 * sin]        y = [y1 | y2], cos / sin of the
//                                                           row's position
// All of it in fp32 from the loaded operands, rounded once to the output type (an eager
// implementation rounds after the norm, the weight and each product).  8-bit rows:
// scale 2^e, e the smallest whole number with max|y| <= 448 * 2^e, codes y * 2^-e rounded to
// the nearest e4m3 (ties to even); a power of two costs no precision and dequantises exactly.
// A row with a non-finite element gets the scale byte 255 (NaN) and zero codes: it reads back
// as NaN.
//
// Bound: HBM for long inputs (each byte read once, written once), a launch and two dependent
// loads (position, cos / sin) for a decode round.  A head row is held by D / 16 lanes, each
// with 8 elements of the first half and their rotation partners of the second, so the
// rotation needs no exchange and the norm (and the 8-bit maximum) is a few shuffles; a lane
// group takes four heads of a token, which keeps enough bytes in flight and reads the
// position, cos / sin and weights once for the four.  16381 tokens of 32 + 8 + 8 bf16 heads,
// 8-bit cache: 78 us, 4.9 TB/s (CTAs of 64 threads fill an SM's registers; with 256, of which
// two fit, 93 us).
#include <algorithm>

#include "common.cuh"

namespace {

__device__ uint32_t g_norm_errors;

constexpr int kThreads = 64;

enum StoreMode { kStoreNone = 0, kStoreSame = 1, kStoreFp8 = 2 };

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, int is64) {
  return is64 ? __ldg(static_cast<const int64_t*>(p) + i)
              : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p) + i));
}

template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

// Weights and cos / sin come in any of the three types.
__device__ __forceinline__ float load_any(const void* p, int64_t i, int dtype) {
  if (dtype == JT_F32) return __ldg(static_cast<const float*>(p) + i);
  if (dtype == JT_BF16) return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
  return __half2float(__ldg(static_cast<const __half*>(p) + i));
}

// Eight consecutive elements as loaded (16 or 32 bytes), 16-byte aligned.
template <typename T>
struct Oct {
  static_assert(sizeof(T) == 2, "16-bit operands");
  uint4 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f<T>(e[i]);
  }
  __device__ __forceinline__ static void store(T* p, const float (&f)[8]) {
    uint4 v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = v;
  }
};
template <>
struct Oct<float> {
  float4 lo, hi;
  __device__ __forceinline__ void load(const float* p) {
    lo = __ldcs(reinterpret_cast<const float4*>(p));
    hi = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void unpack(float (&f)[8]) const {
    f[0] = lo.x; f[1] = lo.y; f[2] = lo.z; f[3] = lo.w;
    f[4] = hi.x; f[5] = hi.y; f[6] = hi.z; f[7] = hi.w;
  }
  __device__ __forceinline__ static void store(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
// Eight weights or cosines of any type.
__device__ __forceinline__ void load_any8(const void* p, int64_t i, int dtype, float (&f)[8]) {
  if (dtype == JT_F32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 a = __ldg(q), b = __ldg(q + 1);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 x = dtype == JT_BF16 ? jt::MmaOp<__nv_bfloat16>::unpack(w[k]) : jt::MmaOp<__half>::unpack(w[k]);
      f[2 * k] = x.x;
      f[2 * k + 1] = x.y;
    }
  }
}

// Scale exponent of an 8-bit row from its largest magnitude (finite): the smallest e with
// amax <= 448 * 2^e, read off the float's fields (448 = 1.75 * 2^8); 0 for a row of zeros,
// at least -127 (e8m0's least exponent, reached only by subnormal rows).
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  if (bits == 0) return 0;
  const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  return max(e, -127);
}
// 2^-e for e in [-127, 120].
__device__ __forceinline__ float exp2_neg(int e) {
  return __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
}
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint2 pack_e4m3x8(const float (&f)[8], float s) {
  return make_uint2(pack_e4m3(f[0] * s, f[1] * s) | (pack_e4m3(f[2] * s, f[3] * s) << 16),
                    pack_e4m3(f[4] * s, f[5] * s) | (pack_e4m3(f[6] * s, f[7] * s) << 16));
}

// Where one row comes from and goes to.
struct Row {
  int64_t token;
  int head;  // within its kind
  int kind;  // 0 query, 1 key, 2 value, -1 none
};
__device__ __forceinline__ Row decode_row(const JtQkNormRopeParams& p, int64_t id, int heads) {
  Row r;
  if (id >= static_cast<int64_t>(p.rows) * heads) {
    r.token = 0;
    r.head = 0;
    r.kind = -1;
    return r;
  }
  r.token = id < 0x7fffffff ? static_cast<int64_t>(static_cast<uint32_t>(id) / static_cast<uint32_t>(heads))
                            : id / heads;
  const int h = static_cast<int>(id - r.token * heads);
  r.kind = h < p.q_heads ? 0 : h < p.q_heads + p.kv_heads ? 1 : 2;
  r.head = r.kind == 0 ? h : r.kind == 1 ? h - p.q_heads : h - p.q_heads - p.kv_heads;
  return r;
}

template <typename T>
__device__ __forceinline__ const T* source_row(const JtQkNormRopeParams& p, const Row& r) {
  if (r.kind == 0) return static_cast<const T*>(p.q) + r.token * p.q_stride0 + r.head * p.q_stride1;
  if (r.kind == 1) return static_cast<const T*>(p.k) + r.token * p.k_stride0 + r.head * p.k_stride1;
  return static_cast<const T*>(p.v) + r.token * p.v_stride0 + r.head * p.v_stride1;
}

// Cache place of a token: page -1 when its slot is negative (skipped) or out of range.
__device__ __forceinline__ void cache_place(const JtQkNormRopeParams& p, int64_t token,
                                            int64_t& page, int64_t& offset) {
  const int64_t slot = load_index(p.slots, token * p.slots_stride, p.slots_is_int64);
  page = -1;
  offset = 0;
  if (slot < 0) return;
  if (slot >= p.num_pages * static_cast<int64_t>(p.page_size)) {
    atomicOr(&g_norm_errors, JT_DEVERR_OUT_OF_RANGE);
    return;
  }
  page = slot < 0x7fffffff
             ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.page_size))
             : slot / p.page_size;
  offset = slot - page * p.page_size;
}

__device__ __forceinline__ int64_t cache_row(const JtQkNormRopeParams& p, int64_t token) {
  int64_t position = load_index(p.positions, token * p.positions_stride, p.positions_is_int64);
  if (position < 0 || position >= p.max_position) {
    atomicOr(&g_norm_errors, JT_DEVERR_OUT_OF_RANGE);
    position = 0;
  }
  return position * p.cache_stride0;
}

// C heads of one kind (0 query, 1 key, 2 value) of one token by a group of D / 16 lanes: all
// their loads first, then row after row.  Position, slot, cos / sin and weights are read once
// for the C rows.
template <typename T, int D, int MODE, int C, int KIND>
__device__ __forceinline__ void norm_unit(const JtQkNormRopeParams& p, int64_t token, int head0,
                                          bool live, int l) {
  constexpr int L = D / 16;
  const int heads = KIND == 0 ? p.q_heads : p.kv_heads;
  const int c1 = 8 * l, c2 = D / 2 + 8 * l;
  const T* src = KIND == 0   ? static_cast<const T*>(p.q) + token * p.q_stride0
                 : KIND == 1 ? static_cast<const T*>(p.k) + token * p.k_stride0
                             : static_cast<const T*>(p.v) + token * p.v_stride0;
  const int64_t head_stride = KIND == 0 ? p.q_stride1 : KIND == 1 ? p.k_stride1 : p.v_stride1;
  Oct<T> x1[C], x2[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const T* row = src + min(head0 + i, heads - 1) * head_stride;
    x1[i].load(row + c1);
    x2[i].load(row + c2);
  }
  int64_t page = -1, offset = 0;
  if (MODE != kStoreNone && KIND >= 1) cache_place(p, token, page, offset);
  float co[8], si[8], w1[8], w2[8];
  if constexpr (KIND < 2) {
    const int64_t cr = cache_row(p, token);
    load_any8(p.cos_sin_cache, cr + c1, p.cache_dtype, co);
    load_any8(p.cos_sin_cache, cr + c2, p.cache_dtype, si);
    const void* weight = KIND == 0 ? p.q_weight : p.k_weight;
    load_any8(weight, c1, p.weight_dtype, w1);
    load_any8(weight, c2, p.weight_dtype, w2);
  }
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int head = head0 + i;
    const bool ok = live && head < heads;
    float a[8], b[8];
    x1[i].unpack(a);
    x2[i].unpack(b);
    if constexpr (KIND < 2) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y1 = a[e] * inv * w1[e];
        const float y2 = b[e] * inv * w2[e];
        a[e] = y1 * co[e] - y2 * si[e];
        b[e] = y2 * co[e] + y1 * si[e];
      }
    }
    if constexpr (MODE == kStoreFp8 && KIND >= 1) {
      // The largest magnitude's bits order like the value, infinities and NaN above all.
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        m = max(m, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (ok && page >= 0) {
        const bool finite = m < 0x7f800000u;
        const int e = finite ? scale_exponent(__uint_as_float(m)) : 0;
        const float s = exp2_neg(e);
        uint8_t* dst = KIND == 1 ? static_cast<uint8_t*>(p.k_pool) + page * p.kp_stride0 +
                                       offset * p.kp_stride1 + head * p.kp_stride2
                                 : static_cast<uint8_t*>(p.v_pool) + page * p.vp_stride0 +
                                       offset * p.vp_stride1 + head * p.vp_stride2;
        *reinterpret_cast<uint2*>(dst + c1) = finite ? pack_e4m3x8(a, s) : make_uint2(0u, 0u);
        *reinterpret_cast<uint2*>(dst + c2) = finite ? pack_e4m3x8(b, s) : make_uint2(0u, 0u);
        if (l == 0) {
          uint8_t* sc = KIND == 1 ? static_cast<uint8_t*>(p.k_scale) + page * p.ks_stride0 +
                                        head * p.ks_stride1 + offset
                                  : static_cast<uint8_t*>(p.v_scale) + page * p.vs_stride0 +
                                        head * p.vs_stride1 + offset;
          *sc = finite ? static_cast<uint8_t>(e + 127) : 255;
        }
      }
    } else {
      T* dst = nullptr;
      if (KIND == 0)
        dst = static_cast<T*>(p.q_out) + token * p.qo_stride0 + head * p.qo_stride1;
      else if (MODE == kStoreNone)
        dst = static_cast<T*>(p.k_out) + token * p.ko_stride0 + head * p.ko_stride1;
      else if (page >= 0)
        dst = KIND == 1 ? static_cast<T*>(p.k_pool) + page * p.kp_stride0 + offset * p.kp_stride1 +
                              head * p.kp_stride2
                        : static_cast<T*>(p.v_pool) + page * p.vp_stride0 + offset * p.vp_stride1 +
                              head * p.vp_stride2;
      if (ok && dst != nullptr) {
        Oct<T>::store(dst + c1, a);  // V: the loaded values, unchanged
        Oct<T>::store(dst + c2, b);
      }
    }
  }
}

template <typename T, int D, int MODE, int C>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const JtQkNormRopeParams p,
                                                                unsigned q_blocks, unsigned k_blocks) {
  constexpr int L = D / 16;              // lanes per row
  constexpr int kGroups = kThreads / L;  // lane groups per CTA
  const int group = threadIdx.x / L, l = threadIdx.x % L;
  // A CTA's rows are of one kind.
  const int kind = blockIdx.x < q_blocks ? 0 : blockIdx.x < q_blocks + k_blocks ? 1 : 2;
  const unsigned block = blockIdx.x - (kind == 0 ? 0u : kind == 1 ? q_blocks : q_blocks + k_blocks);
  const int heads = kind == 0 ? p.q_heads : p.kv_heads;
  const unsigned chunks = (heads + C - 1) / C;
  const uint64_t unit = static_cast<uint64_t>(block) * kGroups + group;
  uint64_t token = unit < 0x80000000u ? static_cast<uint32_t>(unit) / chunks : unit / chunks;
  const int head0 = static_cast<int>(unit - token * chunks) * C;
  const bool live = token < static_cast<uint64_t>(p.rows);
  if (!live) token = p.rows - 1;  // takes part in the shuffles, writes nothing
  if (kind == 0)
    norm_unit<T, D, MODE, C, 0>(p, token, head0, live, l);
  else if (kind == 1)
    norm_unit<T, D, MODE, C, 1>(p, token, head0, live, l);
  else
    norm_unit<T, D, MODE, C, 2>(p, token, head0, live, l);
}

// Any even head dim up to 512 and any alignment: one warp per row, element by element.
template <typename T, int MODE>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_any_kernel(const JtQkNormRopeParams p) {
  constexpr int kPairs = 8;  // rotation pairs per lane: head_dim / 2 <= 256
  const int lane = threadIdx.x & 31, half = p.head_dim / 2;
  const int heads = p.q_heads + p.kv_heads * (MODE == kStoreNone ? 1 : 2);
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  const Row r = decode_row(p, id, heads);
  if (r.kind < 0) return;  // whole warps
  const T* src = source_row<T>(p, r);
  float a[kPairs], b[kPairs];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int d = lane + 32 * i;
    a[i] = d < half ? to_f<T>(src[d]) : 0.f;
    b[i] = d < half ? to_f<T>(src[half + d]) : 0.f;
    ss += a[i] * a[i] + b[i] * b[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  if (r.kind < 2) {
    const float inv = 1.0f / sqrtf(ss / static_cast<float>(p.head_dim) + p.eps);
    const void* w = r.kind == 0 ? p.q_weight : p.k_weight;
    const int64_t cr = cache_row(p, r.token);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      const int d = lane + 32 * i;
      if (d < half) {
        const float y1 = a[i] * inv * load_any(w, d, p.weight_dtype);
        const float y2 = b[i] * inv * load_any(w, half + d, p.weight_dtype);
        const float c = load_any(p.cos_sin_cache, cr + d, p.cache_dtype);
        const float s = load_any(p.cos_sin_cache, cr + half + d, p.cache_dtype);
        a[i] = y1 * c - y2 * s;
        b[i] = y2 * c + y1 * s;
      }
    }
  }
  T* dst = nullptr;
  if (r.kind == 0)
    dst = static_cast<T*>(p.q_out) + r.token * p.qo_stride0 + r.head * p.qo_stride1;
  else if (MODE == kStoreNone)
    dst = static_cast<T*>(p.k_out) + r.token * p.ko_stride0 + r.head * p.ko_stride1;
  if (MODE != kStoreNone && r.kind >= 1) {
    int64_t page, offset;
    cache_place(p, r.token, page, offset);
    if (page < 0) return;
    const int64_t place = r.kind == 1
                              ? page * p.kp_stride0 + offset * p.kp_stride1 + r.head * p.kp_stride2
                              : page * p.vp_stride0 + offset * p.vp_stride1 + r.head * p.vp_stride2;
    if constexpr (MODE == kStoreSame) {
      dst = static_cast<T*>(r.kind == 1 ? p.k_pool : p.v_pool) + place;
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kPairs; ++i)
        m = max(m, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
      m = __reduce_max_sync(0xffffffffu, m);
      const bool finite = m < 0x7f800000u;
      const int e = finite ? scale_exponent(__uint_as_float(m)) : 0;
      const float s = exp2_neg(e);
      uint8_t* codes = static_cast<uint8_t*>(r.kind == 1 ? p.k_pool : p.v_pool) + place;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const int d = lane + 32 * i;
        if (d < half) {
          const uint32_t pair = finite ? pack_e4m3(a[i] * s, b[i] * s) : 0u;
          codes[d] = static_cast<uint8_t>(pair & 0xffu);
          codes[half + d] = static_cast<uint8_t>(pair >> 8);
        }
      }
      if (lane == 0) {
        uint8_t* sc = r.kind == 1 ? static_cast<uint8_t*>(p.k_scale) + page * p.ks_stride0 +
                                        r.head * p.ks_stride1 + offset
                                  : static_cast<uint8_t*>(p.v_scale) + page * p.vs_stride0 +
                                        r.head * p.vs_stride1 + offset;
        *sc = finite ? static_cast<uint8_t>(e + 127) : 255;
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < kPairs; ++i) {
    const int d = lane + 32 * i;
    if (d < half) {
      dst[d] = from_f<T>(a[i]);
      dst[half + d] = from_f<T>(b[i]);
    }
  }
}

bool aligned(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// Eight-element accesses need 16-byte bases and row strides (8 bytes for 8-bit rows).
bool vector_ok(const JtQkNormRopeParams& p) {
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256) return false;
  const int step = p.dtype == JT_F32 ? 4 : 8;
  if (!aligned(p.q, 16) || !aligned(p.k, 16) || !aligned(p.q_out, 16) || !aligned(p.q_weight, 16) ||
      !aligned(p.k_weight, 16) || !aligned(p.cos_sin_cache, 16) ||
      p.cache_stride0 % (p.cache_dtype == JT_F32 ? 4 : 8) != 0 ||
      (p.q_stride0 | p.q_stride1 | p.k_stride0 | p.k_stride1 | p.qo_stride0 | p.qo_stride1) % step != 0)
    return false;
  if (p.store == kStoreNone) return aligned(p.k_out, 16) && (p.ko_stride0 | p.ko_stride1) % step == 0;
  const int pool = p.store == kStoreFp8 ? 8 : 16, pool_step = p.store == kStoreFp8 ? 8 : step;
  return aligned(p.v, 16) && (p.v_stride0 | p.v_stride1) % step == 0 && aligned(p.k_pool, pool) &&
         aligned(p.v_pool, pool) &&
         (p.kp_stride0 | p.kp_stride1 | p.kp_stride2 | p.vp_stride0 | p.vp_stride1 |
          p.vp_stride2) % pool_step == 0;
}

template <typename T, int D, int MODE, int C>
void launch_chunks(const JtQkNormRopeParams& p, cudaStream_t stream) {
  constexpr int kGroups = kThreads / (D / 16);
  auto blocks = [&](int heads) {
    return static_cast<unsigned>((p.rows * ((heads + C - 1) / C) + kGroups - 1) / kGroups);
  };
  const unsigned q = blocks(p.q_heads), k = blocks(p.kv_heads);
  qk_norm_rope_kernel<T, D, MODE, C><<<q + k * (MODE == kStoreNone ? 1 : 2), kThreads, 0, stream>>>(p, q, k);
}

template <typename T, int D, int MODE>
void launch_vector(const JtQkNormRopeParams& p, int64_t rows, int sms, cudaStream_t stream) {
  constexpr int kGroups = kThreads / (D / 16), C = sizeof(T) == 2 ? 4 : 2;
  // C heads per lane group once they still give every SM two CTAs: below that a head each,
  // spread over more SMs, answers sooner.
  if (rows >= 2LL * sms * kGroups * C)
    launch_chunks<T, D, MODE, C>(p, stream);
  else
    launch_chunks<T, D, MODE, 1>(p, stream);
}

template <typename T, int MODE>
void launch_mode(const JtQkNormRopeParams& p, int64_t rows, int sms, cudaStream_t stream) {
  if (vector_ok(p)) {
    if (p.head_dim == 128) return launch_vector<T, 128, MODE>(p, rows, sms, stream);
    if (p.head_dim == 64) return launch_vector<T, 64, MODE>(p, rows, sms, stream);
    return launch_vector<T, 256, MODE>(p, rows, sms, stream);
  }
  const int64_t grid = (rows + kThreads / 32 - 1) / (kThreads / 32);
  qk_norm_rope_any_kernel<T, MODE><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
}

template <typename T>
void launch_type(const JtQkNormRopeParams& p, int64_t rows, int sms, cudaStream_t stream) {
  if (p.store == kStoreNone) return launch_mode<T, kStoreNone>(p, rows, sms, stream);
  if (p.store == kStoreSame) return launch_mode<T, kStoreSame>(p, rows, sms, stream);
  launch_mode<T, kStoreFp8>(p, rows, sms, stream);
}

bool known_dtype(int d) { return d == JT_BF16 || d == JT_F16 || d == JT_F32; }

}  // namespace

int jt_read_errors_norm(uint32_t* bits) {
  uint32_t zero = 0;
  int rc = jt_cuda_check(cudaMemcpyFromSymbol(bits, g_norm_errors, sizeof(uint32_t)),
                         "read norm error word");
  if (rc != JT_OK) return rc;
  return jt_cuda_check(cudaMemcpyToSymbol(g_norm_errors, &zero, sizeof(uint32_t)),
                       "clear norm error word");
}

extern "C" int jt_qk_norm_rope_launch(const JtQkNormRopeParams* p, cudaStream_t stream) {
  if (p == nullptr) return jt_fail(JT_ERR_INVALID, "qk_norm_rope: null params");
  if (p->rows < 0 || p->q_heads < 1 || p->kv_heads < 1 || p->head_dim < 2 || p->head_dim % 2 != 0 ||
      p->head_dim > 512 || p->max_position < 1)
    return jt_fail(JT_ERR_INVALID, "qk_norm_rope: invalid geometry");
  if (p->store < kStoreNone || p->store > kStoreFp8 ||
      (p->store != kStoreNone && (p->page_size < 1 || p->num_pages < 1)))
    return jt_fail(JT_ERR_INVALID, "qk_norm_rope: invalid cache geometry");
  if (!known_dtype(p->dtype) || !known_dtype(p->weight_dtype) || !known_dtype(p->cache_dtype))
    return jt_fail(JT_ERR_UNSUPPORTED, "qk_norm_rope: operands must be bf16, f16 or f32");
  if (p->rows == 0) return JT_OK;
  if (!p->q || !p->k || !p->q_weight || !p->k_weight || !p->positions || !p->cos_sin_cache ||
      !p->q_out || (p->store == kStoreNone && !p->k_out) ||
      (p->store != kStoreNone && (!p->v || !p->slots || !p->k_pool || !p->v_pool)) ||
      (p->store == kStoreFp8 && (!p->k_scale || !p->v_scale)))
    return jt_fail(JT_ERR_INVALID, "qk_norm_rope: null tensor pointer");
  const int64_t heads =
      static_cast<int64_t>(p->q_heads) + static_cast<int64_t>(p->kv_heads) * (p->store == kStoreNone ? 1 : 2);
  const int64_t rows = p->rows * heads;
  if (heads > 0x7fffffff || rows / 8 >= 0x7fffffff)
    return jt_fail(JT_ERR_INVALID, "qk_norm_rope: too many rows");
  int dev = 0, sms = 0;
  int rc = jt_cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc != JT_OK) return rc;
  rc = jt_cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev),
                     "SM count");
  if (rc != JT_OK) return rc;
  if (p->dtype == JT_BF16)
    launch_type<__nv_bfloat16>(*p, rows, sms, stream);
  else if (p->dtype == JT_F16)
    launch_type<__half>(*p, rows, sms, stream);
  else
    launch_type<float>(*p, rows, sms, stream);
  return jt_cuda_check(cudaGetLastError(), "qk_norm_rope launch");
}
