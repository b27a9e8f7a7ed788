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
// loads (position, cos / sin) for a decode round.  A head row is held by D / 8 lanes, each
// with 4 elements of the first half and their rotation partners of the second, so the
// rotation needs no exchange and the norm (and the 8-bit maximum) is a few shuffles; a lane
// group loads kRows rows before it computes any, to keep enough bytes in flight.
#include <algorithm>

#include "common.cuh"

namespace {

__device__ uint32_t g_norm_errors;

constexpr int kThreads = 256;

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

// Four consecutive elements as loaded (8 or 16 bytes).
template <typename T>
struct Quad {
  static_assert(sizeof(T) == 2, "16-bit operands");
  uint2 raw;
  __device__ __forceinline__ void load(const T* p) { raw = __ldcs(reinterpret_cast<const uint2*>(p)); }
  __device__ __forceinline__ void unpack(float (&f)[4]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = to_f<T>(e[i]);
  }
  __device__ __forceinline__ static void store(T* p, const float (&f)[4]) {
    uint2 v;
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint2*>(p) = v;
  }
};
template <>
struct Quad<float> {
  float4 raw;
  __device__ __forceinline__ void load(const float* p) { raw = __ldcs(reinterpret_cast<const float4*>(p)); }
  __device__ __forceinline__ void unpack(float (&f)[4]) const {
    f[0] = raw.x; f[1] = raw.y; f[2] = raw.z; f[3] = raw.w;
  }
  __device__ __forceinline__ static void store(float* p, const float (&f)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};

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
__device__ __forceinline__ uint32_t pack_e4m3x4(const float (&f)[4], float s) {
  return pack_e4m3(f[0] * s, f[1] * s) | (pack_e4m3(f[2] * s, f[3] * s) << 16);
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

template <typename T, int D, int MODE, int kRows>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const JtQkNormRopeParams p) {
  constexpr int L = D / 8;                  // lanes per row
  constexpr int kGroups = kThreads / L;     // lane groups per CTA
  const int group = threadIdx.x / L, l = threadIdx.x % L;
  const int heads = p.q_heads + p.kv_heads * (MODE == kStoreNone ? 1 : 2);
  const int64_t base = static_cast<int64_t>(blockIdx.x) * (kGroups * kRows) + group;
  const int c1 = 4 * l, c2 = D / 2 + 4 * l;

  Row row[kRows];
  Quad<T> x1[kRows], x2[kRows];
  float4 co[kRows], si[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    row[i] = decode_row(p, base + i * kGroups, heads);
    if (row[i].kind >= 0) {
      const T* src = source_row<T>(p, row[i]);
      x1[i].load(src + c1);
      x2[i].load(src + c2);
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    co[i] = make_float4(1.f, 1.f, 1.f, 1.f);
    si[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row[i].kind == 0 || row[i].kind == 1) {
      const int64_t cr = cache_row(p, row[i].token);
      if (p.cache_dtype == JT_F32) {
        const float* c = static_cast<const float*>(p.cos_sin_cache) + cr;
        co[i] = __ldg(reinterpret_cast<const float4*>(c + c1));
        si[i] = __ldg(reinterpret_cast<const float4*>(c + c2));
      } else {
        co[i] = make_float4(load_any(p.cos_sin_cache, cr + c1, p.cache_dtype),
                            load_any(p.cos_sin_cache, cr + c1 + 1, p.cache_dtype),
                            load_any(p.cos_sin_cache, cr + c1 + 2, p.cache_dtype),
                            load_any(p.cos_sin_cache, cr + c1 + 3, p.cache_dtype));
        si[i] = make_float4(load_any(p.cos_sin_cache, cr + c2, p.cache_dtype),
                            load_any(p.cos_sin_cache, cr + c2 + 1, p.cache_dtype),
                            load_any(p.cos_sin_cache, cr + c2 + 2, p.cache_dtype),
                            load_any(p.cos_sin_cache, cr + c2 + 3, p.cache_dtype));
      }
    }
  }
  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    wq[e] = load_any(p.q_weight, c1 + e, p.weight_dtype);
    wq[4 + e] = load_any(p.q_weight, c2 + e, p.weight_dtype);
    wk[e] = load_any(p.k_weight, c1 + e, p.weight_dtype);
    wk[4 + e] = load_any(p.k_weight, c2 + e, p.weight_dtype);
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const Row& r = row[i];
    float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
    if (r.kind >= 0) {
      x1[i].unpack(a);
      x2[i].unpack(b);
    }
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (r.kind == 0 || r.kind == 1) {
      const float inv = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
      const float c[4] = {co[i].x, co[i].y, co[i].z, co[i].w};
      const float s[4] = {si[i].x, si[i].y, si[i].z, si[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float y1 = a[e] * inv * (r.kind == 0 ? wq[e] : wk[e]);
        const float y2 = b[e] * inv * (r.kind == 0 ? wq[4 + e] : wk[4 + e]);
        a[e] = y1 * c[e] - y2 * s[e];
        b[e] = y2 * c[e] + y1 * s[e];
      }
    }
    if constexpr (MODE == kStoreFp8) {
      // The largest magnitude's bits order like the value, infinities and NaN above all.
      uint32_t m = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        m = max(m, max(__float_as_uint(a[e]) & 0x7fffffffu, __float_as_uint(b[e]) & 0x7fffffffu));
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (r.kind >= 1) {
        int64_t page, offset;
        cache_place(p, r.token, page, offset);
        if (page >= 0) {
          const bool is_k = r.kind == 1;
          const bool finite = m < 0x7f800000u;
          const int e = finite ? scale_exponent(__uint_as_float(m)) : 0;
          const float s = exp2_neg(e);
          uint8_t* dst = is_k ? static_cast<uint8_t*>(p.k_pool) + page * p.kp_stride0 +
                                    offset * p.kp_stride1 + r.head * p.kp_stride2
                              : static_cast<uint8_t*>(p.v_pool) + page * p.vp_stride0 +
                                    offset * p.vp_stride1 + r.head * p.vp_stride2;
          *reinterpret_cast<uint32_t*>(dst + c1) = finite ? pack_e4m3x4(a, s) : 0u;
          *reinterpret_cast<uint32_t*>(dst + c2) = finite ? pack_e4m3x4(b, s) : 0u;
          if (l == 0) {
            uint8_t* sc = is_k ? static_cast<uint8_t*>(p.k_scale) + page * p.ks_stride0 +
                                     r.head * p.ks_stride1 + offset
                               : static_cast<uint8_t*>(p.v_scale) + page * p.vs_stride0 +
                                     r.head * p.vs_stride1 + offset;
            *sc = finite ? static_cast<uint8_t>(e + 127) : 255;
          }
        }
      }
    }
    if (r.kind == 0) {
      T* dst = static_cast<T*>(p.q_out) + r.token * p.qo_stride0 + r.head * p.qo_stride1;
      Quad<T>::store(dst + c1, a);
      Quad<T>::store(dst + c2, b);
    } else if (MODE == kStoreNone && r.kind == 1) {
      T* dst = static_cast<T*>(p.k_out) + r.token * p.ko_stride0 + r.head * p.ko_stride1;
      Quad<T>::store(dst + c1, a);
      Quad<T>::store(dst + c2, b);
    } else if (MODE == kStoreSame && r.kind >= 1) {
      int64_t page, offset;
      cache_place(p, r.token, page, offset);
      if (page >= 0) {
        T* dst = r.kind == 1 ? static_cast<T*>(p.k_pool) + page * p.kp_stride0 +
                                   offset * p.kp_stride1 + r.head * p.kp_stride2
                             : static_cast<T*>(p.v_pool) + page * p.vp_stride0 +
                                   offset * p.vp_stride1 + r.head * p.vp_stride2;
        Quad<T>::store(dst + c1, a);  // V: the loaded values, unchanged
        Quad<T>::store(dst + c2, b);
      }
    }
  }
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

// Four-element accesses need bases and row strides on four elements (16 bytes for the fp32
// cos / sin cache; four bytes for 8-bit rows).
bool vector_ok(const JtQkNormRopeParams& p) {
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256) return false;
  const int quad = p.dtype == JT_F32 ? 16 : 8;
  if (!aligned(p.q, quad) || !aligned(p.k, quad) || !aligned(p.q_out, quad) ||
      (p.q_stride0 | p.q_stride1 | p.k_stride0 | p.k_stride1 | p.qo_stride0 | p.qo_stride1) % 4 != 0)
    return false;
  if (p.cache_dtype == JT_F32 && (!aligned(p.cos_sin_cache, 16) || p.cache_stride0 % 4 != 0))
    return false;
  if (p.store == kStoreNone)
    return aligned(p.k_out, quad) && (p.ko_stride0 | p.ko_stride1) % 4 == 0;
  const int pool = p.store == kStoreFp8 ? 4 : quad;
  return aligned(p.v, quad) && (p.v_stride0 | p.v_stride1) % 4 == 0 && aligned(p.k_pool, pool) &&
         aligned(p.v_pool, pool) &&
         (p.kp_stride0 | p.kp_stride1 | p.kp_stride2 | p.vp_stride0 | p.vp_stride1 |
          p.vp_stride2) % 4 == 0;
}

template <typename T, int D, int MODE>
void launch_vector(const JtQkNormRopeParams& p, int64_t rows, int sms, cudaStream_t stream) {
  constexpr int kGroups = kThreads / (D / 8);
  // Four rows per lane group once they still give every SM two CTAs: below that a row each,
  // spread over more SMs, answers sooner.
  if (rows >= 2LL * sms * kGroups * 4) {
    const int64_t grid = (rows + kGroups * 4 - 1) / (kGroups * 4);
    qk_norm_rope_kernel<T, D, MODE, 4><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
  } else {
    const int64_t grid = (rows + kGroups - 1) / kGroups;
    qk_norm_rope_kernel<T, D, MODE, 1><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
  }
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
