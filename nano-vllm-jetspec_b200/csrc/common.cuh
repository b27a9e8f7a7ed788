// Shared helpers for the sm_100a JetSpec kernels: status plumbing, 16-byte async
// copies, ldmatrix and the bf16/f16 warp-level MMA used by the v0 attention core.
#pragma once

#include <cuda_runtime.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/jetspec_b200.h"

// ---- host-side status -------------------------------------------------------------
// Defined in api.cu; records a one-line message for jt_last_error() and returns code.
int jt_fail(int code, const char* fmt, ...);
int jt_cuda_check(cudaError_t err, const char* what);

// Per-translation-unit device error word readers (each TU owns its own word).
int jt_read_errors_kv(uint32_t* bits);
int jt_read_errors_attn(uint32_t* bits);
int jt_read_errors_rope(uint32_t* bits);
int jt_read_errors_accept(uint32_t* bits);
int jt_read_errors_meta(uint32_t* bits);
int jt_read_errors_rowlin(uint32_t* bits);
int jt_read_errors_f32(uint32_t* bits);
int jt_read_errors_maps(uint32_t* bits);
int jt_read_errors_norm(uint32_t* bits);
int jt_read_errors_fp8_commit(uint32_t* bits);
int jt_read_errors_attn_fp8(uint32_t* bits);

// fp32-operand tree attention (tree_attn_f32.cu), for parameters the entry point checked.
int jt_tree_attn_f32_launch(const JtTreeAttnParams& p, cudaStream_t stream);

#define JT_DEVERR_OUT_OF_RANGE 1u
#define JT_DEVERR_TREE_TOO_LARGE 2u
#define JT_DEVERR_TIMEOUT 4u

// ---- device helpers ----------------------------------------------------------------
namespace jt {

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16-byte global->shared copy; src_bytes == 0 zero-fills the destination.
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src),
               "r"(src_bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N));
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

template <typename T>
struct MmaOp;

template <>
struct MmaOp<__nv_bfloat16> {
  __device__ __forceinline__ static void run(float c[4], const uint32_t a[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // Round two fp32 values to the operand type and pack (low half = first value).
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&v));
  }
};

template <>
struct MmaOp<__half> {
  __device__ __forceinline__ static void run(float c[4], const uint32_t a[4], uint32_t b0,
                                             uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __device__ __forceinline__ static float2 unpack(uint32_t v) {
    return __half22float2(*reinterpret_cast<__half2*>(&v));
  }
};

__device__ __forceinline__ float fast_exp2(float x) {
  // ex2.approx of -inf is +0, which the online softmax relies on for masked keys.
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace jt
