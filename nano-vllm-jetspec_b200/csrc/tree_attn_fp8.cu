// Packed tree attention over an 8-bit paged cache (e4m3 codes, power-of-two row scales).
//
// For query row i (node j, head hq) of request r: keys are positions 0..P+T-1 (prefix pages,
// then the T tree nodes), visible when the position is below P, or is node n <= j with zero
// bias.  s = scale * sum_d q_d k_d, p = exp(s - max), out = sum p v / sum p, with
// k = code * 2^(kbyte - 127) and v likewise.
#include "common.cuh"

#include <cuda_fp8.h>

namespace {

__device__ uint32_t g_attn_fp8_errors;

constexpr int kThreads = 128;

__device__ __forceinline__ float code_value(uint8_t c) {
  __nv_fp8_e4m3 v;
  v.__x = c;
  return static_cast<float>(v);
}
// 2^(byte - 127); byte 255 is NaN, byte 0 the subnormal 2^-127.
__device__ __forceinline__ float scale_value(uint8_t b) {
  if (b == 255) return __uint_as_float(0x7fc00000u);
  return b == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(static_cast<uint32_t>(b) << 23);
}

// One CTA per (packed node, query head): 128 keys at a time, a score per thread, then an
// output element per thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) tree_attn_fp8_kernel(const JtTreeAttnFp8Params p) {
  __shared__ float sq[128], prob[kThreads], red[kThreads / 32];
  __shared__ int64_t place[kThreads], vplace[kThreads];
  const int node = blockIdx.x, hq = blockIdx.y, h = hq / p.groups, tid = threadIdx.x;
  const int r = p.query_to_request[node], j = p.query_local_row[node];
  const int P = max(p.prefix_lens[r], 0), T_r = p.node_counts[r], q0 = p.cu_seqlens_q[r];
  if (T_r > 1024) {
    if (tid == 0) atomicOr(&g_attn_fp8_errors, JT_DEVERR_TREE_TOO_LARGE);
    return;
  }
  const int D = p.head_dim;
  const T* q = static_cast<const T*>(p.q) + node * p.q_stride0 + hq * p.q_stride1;
  if (tid < D) sq[tid] = static_cast<float>(q[tid]);
  __syncthreads();
  const int32_t* table = p.block_tables + r * p.table_stride0;
  const float* bias = p.qq_bias + p.qq_bias_offsets[r] + static_cast<int64_t>(j) * T_r;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  for (int k0 = 0; k0 < P + j + 1; k0 += kThreads) {
    const int pos = k0 + tid;
    int64_t slot = -1;
    if (pos < P) {
      const int col = pos / p.block_size;
      if (col < p.table_width) slot = static_cast<int64_t>(table[col]) * p.block_size + pos % p.block_size;
    } else if (pos <= P + j && bias[pos - P] == 0.f) {
      slot = p.tree_slots[q0 + pos - P];
    }
    const bool want = pos < P || (pos <= P + j && bias[pos - P] == 0.f);
    if (slot < 0 || slot >= p.num_blocks * p.block_size) {
      if (want) atomicOr(&g_attn_fp8_errors, JT_DEVERR_OUT_OF_RANGE);
      slot = -1;
    }
    float s = -INFINITY, vf = 0.f;
    place[tid] = -1;
    if (slot >= 0) {
      const int64_t page = slot / p.block_size, off = slot % p.block_size;
      const uint8_t* k = static_cast<const uint8_t*>(p.k_pool) + page * p.k_stride0 +
                         off * p.k_stride1 + h * p.k_stride2;
      s = 0.f;
      for (int d = 0; d < D; ++d) s += sq[d] * code_value(k[d]);
      s *= scale_value(static_cast<const uint8_t*>(p.k_scale)[page * p.ks_stride0 + h * p.ks_stride1 + off]);
      s *= p.scale;
      vf = scale_value(static_cast<const uint8_t*>(p.v_scale)[page * p.vs_stride0 + h * p.vs_stride1 + off]);
      place[tid] = page * p.v_stride0 + off * p.v_stride1 + h * p.v_stride2;
    }
    float mx = s;
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((tid & 31) == 0) red[tid >> 5] = mx;
    __syncthreads();
    const float top = fmaxf(fmaxf(red[0], red[1]), fmaxf(fmaxf(red[2], red[3]), m));
    const float ref = top == -INFINITY ? 0.f : top;
    const float w = slot >= 0 ? expf(s - ref) : 0.f;
    const float keep = m == -INFINITY ? 0.f : expf(m - ref);
    m = top;
    float sum = w;
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = sum;
    prob[tid] = w * vf;
    __syncthreads();
    l = l * keep + (red[0] + red[1] + red[2] + red[3]);
    acc *= keep;
    if (tid < D)
      for (int i = 0; i < kThreads; ++i)
        if (place[i] >= 0)
          acc += prob[i] * code_value(static_cast<const uint8_t*>(p.v_pool)[place[i] + tid]);
    __syncthreads();
  }
  if (tid < D) {
    const float o = l == 0.f ? 0.f : acc / l;
    const int64_t at = node * p.out_stride0 + hq * p.out_stride1 + tid;
    if (p.out_dtype == JT_F32)
      static_cast<float*>(p.out)[at] = o;
    else
      static_cast<T*>(p.out)[at] = T(o);
  }
}

}  // namespace

int jt_read_errors_attn_fp8(uint32_t* bits) {
  uint32_t zero = 0;
  int rc = jt_cuda_check(cudaMemcpyFromSymbol(bits, g_attn_fp8_errors, sizeof(uint32_t)),
                         "read fp8 attention error word");
  if (rc != JT_OK) return rc;
  return jt_cuda_check(cudaMemcpyToSymbol(g_attn_fp8_errors, &zero, sizeof(uint32_t)),
                       "clear fp8 attention error word");
}

extern "C" int64_t jt_tree_attn_fp8_workspace_size(int32_t num_requests, int32_t total_queries,
                                                   int32_t num_kv_heads, int32_t groups,
                                                   int32_t head_dim) {
  if (num_requests < 1 || total_queries < 1 || num_kv_heads < 1 || groups < 1 || head_dim < 1)
    return -1;
  return 0;
}

extern "C" int jt_tree_attn_fp8_launch(const JtTreeAttnFp8Params* p, cudaStream_t stream) {
  if (p == nullptr) return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: null params");
  if (p->num_requests < 1 || p->total_queries < 1 || p->num_kv_heads < 1 || p->groups < 1 ||
      p->groups > 128 || p->block_size < 1 || p->num_blocks < 1 || p->table_width < 1)
    return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: invalid geometry");
  if (p->head_dim < 16 || p->head_dim > 128 || p->head_dim % 16 != 0)
    return jt_fail(JT_ERR_UNSUPPORTED, "tree_attn_fp8: head_dim %d is not a multiple of 16 up to 128",
                   p->head_dim);
  if (p->dtype != JT_BF16 && p->dtype != JT_F16)
    return jt_fail(JT_ERR_UNSUPPORTED, "tree_attn_fp8: queries must be bf16 or f16");
  if (p->out_dtype != p->dtype && p->out_dtype != JT_F32)
    return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: output dtype must match the queries or be f32");
  if (!(p->scale > 0.f) || p->scale > 3.0e38f)
    return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: the scale must be positive and finite");
  if (!p->out || !p->q || !p->k_pool || !p->v_pool || !p->k_scale || !p->v_scale ||
      !p->cu_seqlens_q || !p->query_to_request || !p->query_local_row || !p->prefix_lens ||
      !p->node_counts || !p->block_tables || !p->tree_slots || !p->qq_bias || !p->qq_bias_offsets)
    return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: null tensor pointer");
  const dim3 grid(p->total_queries, p->num_kv_heads * p->groups);
  if (p->dtype == JT_BF16)
    tree_attn_fp8_kernel<__nv_bfloat16><<<grid, kThreads, 0, stream>>>(*p);
  else
    tree_attn_fp8_kernel<__half><<<grid, kThreads, 0, stream>>>(*p);
  return jt_cuda_check(cudaGetLastError(), "tree_attn_fp8 launch");
}
