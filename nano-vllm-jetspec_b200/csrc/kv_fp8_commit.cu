// Accepted-only commit of an 8-bit cache: e4m3 rows and their scales in one launch.
//
//   kv_pool [2, L, blocks, B, H, D] codes:   row dst <- row src   (every axis, layer, head)
//   kv_scale [2, L, blocks, H, B] bytes:     dst <- src
// A pure copy with every read of a plane before any write to it, so that overlapping slot
// sets behave like a gather followed by a scatter.  A plane is one (axis, layer, head, chunk
// of W 16-byte words of the head row) over every slot; one CTA gathers it into shared memory,
// synchronises and scatters it.  Planes cover disjoint bytes: no CTA waits for another.
//
// Bound: HBM (each 32-byte sector read and written once: W >= 2 keeps sectors whole), and for
// small rounds the launch and two dependent loads (slot, row).
#include <algorithm>

#include "common.cuh"

namespace {

__device__ uint32_t g_fp8_commit_errors;

constexpr int kThreads = 256;
constexpr int kUnroll = 4;
constexpr int kSmemCap = 200 * 1024;
// A wider chunk is taken while the staging stays below this, so that several CTAs share an
// SM and one's gather overlaps another's scatter.
constexpr int kSmemShare = 72 * 1024;

__device__ __forceinline__ int64_t load_slot(const void* base, int is64, int64_t i) {
  return is64 ? __ldg(static_cast<const int64_t*>(base) + i)
              : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(base) + i));
}

struct Place {
  int64_t page, offset;
  bool ok;
};
__device__ __forceinline__ Place place(const JtKvFp8CommitParams& p, const void* slots, int s) {
  const int64_t slot = load_slot(slots, p.slot_is_int64, s);
  Place r;
  r.ok = slot >= 0 && slot < p.num_blocks * static_cast<int64_t>(p.block_size);
  if (slot >= 0 && slot < 0x7fffffff) {  // 32-bit division for every pool in use
    r.page = static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.block_size);
  } else {
    r.page = slot / p.block_size;
  }
  r.offset = slot - r.page * p.block_size;
  return r;
}

template <int W>
__global__ void __launch_bounds__(kThreads) kv_fp8_commit_kernel(const JtKvFp8CommitParams p,
                                                                 int planes, int chunks) {
  extern __shared__ __align__(16) int4 staging[];
  const int n = p.num_slots, units = n * W;
  uint8_t* bytes = reinterpret_cast<uint8_t*>(staging + units);
  for (int plane = blockIdx.x; plane < planes; plane += gridDim.x) {
    const int chunk = plane % chunks;
    int rest = plane / chunks;
    const int head = rest % p.num_kv_heads;
    rest /= p.num_kv_heads;
    const int layer = rest % p.num_layers, axis = rest / p.num_layers;
    char* rows = static_cast<char*>(p.kv_pool) + axis * p.stride_axis + layer * p.stride_layer +
                 head * p.stride_head + chunk * (W * 16);
    uint8_t* scales = static_cast<uint8_t*>(p.kv_scale) + axis * p.scale_axis +
                      layer * p.scale_layer + head * p.scale_head;
    for (int base = threadIdx.x; base < units; base += kThreads * kUnroll) {
      int4 v[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) {
        const int i = base + k * kThreads;
        v[k] = make_int4(0, 0, 0, 0);
        if (i < units) {
          const Place s = place(p, p.source_slots, i / W);
          if (s.ok)
            v[k] = *reinterpret_cast<const int4*>(rows + s.page * p.stride_block +
                                                  s.offset * p.stride_offset + (i % W) * 16);
        }
      }
#pragma unroll
      for (int k = 0; k < kUnroll; ++k)
        if (base + k * kThreads < units) staging[base + k * kThreads] = v[k];
    }
    if (chunk == 0)
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const Place s = place(p, p.source_slots, i);
        if (s.ok)
          bytes[i] = scales[s.page * p.scale_block + s.offset];
        else
          atomicOr(&g_fp8_commit_errors, JT_DEVERR_OUT_OF_RANGE);
      }
    __syncthreads();  // every read of this plane precedes every write to it
    for (int i = threadIdx.x; i < units; i += kThreads) {
      const Place s = place(p, p.source_slots, i / W), d = place(p, p.destination_slots, i / W);
      if (s.ok && d.ok)
        *reinterpret_cast<int4*>(rows + d.page * p.stride_block + d.offset * p.stride_offset +
                                 (i % W) * 16) = staging[i];
    }
    if (chunk == 0)
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const Place s = place(p, p.source_slots, i), d = place(p, p.destination_slots, i);
        if (s.ok && d.ok)
          scales[d.page * p.scale_block + d.offset] = bytes[i];
        else if (!d.ok)
          atomicOr(&g_fp8_commit_errors, JT_DEVERR_OUT_OF_RANGE);
      }
    __syncthreads();  // the staging is free for the next plane
  }
}

template <int W>
int launch(const JtKvFp8CommitParams& p, int sms, cudaStream_t stream) {
  const int chunks = p.head_dim / (16 * W);
  const int64_t planes = 2LL * p.num_layers * p.num_kv_heads * chunks;
  if (planes > 0x7fffffff) return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: too many planes");
  const int smem = p.num_slots * (W * 16 + 1);
  int rc = jt_cuda_check(cudaFuncSetAttribute(kv_fp8_commit_kernel<W>,
                                              cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap),
                         "kv_fp8_commit smem attribute");
  if (rc != JT_OK) return rc;
  const int grid = static_cast<int>(std::min<int64_t>(planes, 16LL * sms));
  kv_fp8_commit_kernel<W><<<grid, kThreads, smem, stream>>>(p, static_cast<int>(planes), chunks);
  return jt_cuda_check(cudaGetLastError(), "kv_fp8_commit launch");
}

}  // namespace

int jt_read_errors_fp8_commit(uint32_t* bits) {
  uint32_t zero = 0;
  int rc = jt_cuda_check(cudaMemcpyFromSymbol(bits, g_fp8_commit_errors, sizeof(uint32_t)),
                         "read fp8 commit error word");
  if (rc != JT_OK) return rc;
  return jt_cuda_check(cudaMemcpyToSymbol(g_fp8_commit_errors, &zero, sizeof(uint32_t)),
                       "clear fp8 commit error word");
}

extern "C" int32_t jt_kv_fp8_commit_max_slots(void) { return kSmemCap / 17; }

extern "C" int jt_kv_fp8_commit_launch(const JtKvFp8CommitParams* p, cudaStream_t stream) {
  if (p == nullptr) return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: null params");
  if (p->num_slots < 0 || p->num_layers < 1 || p->num_kv_heads < 1 || p->head_dim < 16 ||
      p->head_dim % 16 != 0 || p->block_size < 1 || p->num_blocks < 1)
    return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: invalid geometry");
  if (p->num_slots == 0) return JT_OK;
  if (p->num_slots > jt_kv_fp8_commit_max_slots())
    return jt_fail(JT_ERR_UNSUPPORTED, "kv_fp8_commit: %d slots exceed the per-call limit of %d",
                   p->num_slots, jt_kv_fp8_commit_max_slots());
  if (!p->kv_pool || !p->kv_scale || !p->source_slots || !p->destination_slots)
    return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(p->kv_pool) & 15u) != 0 ||
      (p->stride_axis | p->stride_layer | p->stride_block | p->stride_offset | p->stride_head) % 16 != 0)
    return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: rows must be 16-byte aligned");
  int dev = 0, sms = 0;
  int rc = jt_cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc != JT_OK) return rc;
  rc = jt_cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev),
                     "SM count");
  if (rc != JT_OK) return rc;
  const int words = p->head_dim / 16;
  const int64_t n = p->num_slots;
  for (int w : {8, 4, 2})
    if (words % w == 0 && n * (w * 16 + 1) <= kSmemShare)
      return w == 8 ? launch<8>(*p, sms, stream)
                    : w == 4 ? launch<4>(*p, sms, stream) : launch<2>(*p, sms, stream);
  return launch<1>(*p, sms, stream);
}
