// Accepted-only commit of an 8-bit cache: e4m3 rows and their scales in one launch.
//
//   kv_pool [2, L, blocks, B, H, D] codes:   row dst <- row src   (every axis, layer, head)
//   kv_scale [2, L, blocks, H, B] bytes:     dst <- src
// A pure copy with every read of a plane before any write to it, so that overlapping slot
// sets behave like a gather followed by a scatter.  A plane is one (axis, layer, head, chunk
// of W 16-byte words of the head row) over every slot; a CTA, or for many slots a cluster of
// CTAs with a part of the slots each, gathers it into shared memory, meets at the cluster's
// barrier and scatters it.  Planes cover disjoint bytes: no cluster waits for another.
//
// Bound: HBM, and for small rounds the launch and two dependent loads (slot, row).  Whole 128-byte
// rows are read and written once, but a scale byte moves a 32-byte sector each way: 2000 slots of
// 36 layers and 8 heads are 297 MB of payload and 74 MB more of such sectors, in 65 us 5.7 TB/s.  The rows are gathered by cp.async, a plane in flight at a
// time, and a CTA's staging is kept below 40 KB so that several share an SM and one's gather
// overlaps another's scatter.
#include <algorithm>

#include "common.cuh"

namespace {

__device__ uint32_t g_fp8_commit_errors;

constexpr int kThreads = 256;
constexpr int kSmemCap = 220 * 1024;
constexpr int kSmemShare = 40 * 1024;
constexpr int kMaxCluster = 8;
constexpr int kSlotBytes = 17;  // (page, offset) of source and destination, the scale byte
constexpr int kMaxSlots = 200 * 1024 / 17;
static_assert((kMaxSlots + kMaxCluster - 1) / kMaxCluster * (8 * 16 + kSlotBytes) <= kSmemCap,
              "the largest cluster stages every slot");

__device__ __forceinline__ int64_t load_slot(const void* base, int is64, int64_t i) {
  return is64 ? __ldg(static_cast<const int64_t*>(base) + i)
              : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(base) + i));
}

// Page and offset of a slot, page -1 outside the pool.
__device__ __forceinline__ int2 place(const JtKvFp8CommitParams& p, const void* slots, int s) {
  const int64_t slot = load_slot(slots, p.slot_is_int64, s);
  if (slot < 0 || slot >= p.num_blocks * static_cast<int64_t>(p.block_size)) {
    atomicOr(&g_fp8_commit_errors, JT_DEVERR_OUT_OF_RANGE);
    return make_int2(-1, 0);
  }
  // 32-bit division for every pool in use.
  const int64_t page = slot < 0x7fffffff
                           ? static_cast<int64_t>(static_cast<uint32_t>(slot) / static_cast<uint32_t>(p.block_size))
                           : slot / p.block_size;
  return make_int2(static_cast<int>(page), static_cast<int>(slot - page * p.block_size));
}

template <int W>
__global__ void __launch_bounds__(kThreads) kv_fp8_commit_kernel(const JtKvFp8CommitParams p,
                                                                 int planes, int chunks, int per) {
  extern __shared__ __align__(16) int4 staging[];  // [per][W], then [per] places, [per] bytes
  int4* places = staging + per * W;                // source page, offset, destination page, offset
  uint8_t* bytes = reinterpret_cast<uint8_t*>(places + per);
  uint32_t rank, cluster;
  asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctaid.x;\n" : "=r"(cluster));
  const int lo = static_cast<int>(rank) * per, n = max(0, min(per, p.num_slots - lo));
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int2 s = place(p, p.source_slots, lo + i), d = place(p, p.destination_slots, lo + i);
    const bool ok = s.x >= 0 && d.x >= 0;
    places[i] = make_int4(ok ? s.x : -1, s.y, d.x, d.y);
  }
  __syncthreads();
  for (int plane = blockIdx.x / cluster; plane < planes; plane += gridDim.x / cluster) {
    const int chunk = plane % chunks;
    int rest = plane / chunks;
    const int head = rest % p.num_kv_heads;
    rest /= p.num_kv_heads;
    const int layer = rest % p.num_layers, axis = rest / p.num_layers;
    char* rows = static_cast<char*>(p.kv_pool) + axis * p.stride_axis + layer * p.stride_layer +
                 head * p.stride_head + chunk * (W * 16);
    uint8_t* scales = static_cast<uint8_t*>(p.kv_scale) + axis * p.scale_axis +
                      layer * p.scale_layer + head * p.scale_head;
    for (int i = threadIdx.x; i < n * W; i += kThreads) {
      const int4 at = places[i / W];
      if (at.x >= 0)
        jt::cp_async_16(jt::smem_u32(staging + i),
                        rows + at.x * p.stride_block + at.y * p.stride_offset + (i % W) * 16, 16);
    }
    if (chunk == 0)
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const int4 at = places[i];
        if (at.x >= 0) bytes[i] = scales[at.x * p.scale_block + at.y];
      }
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    // Every read of this plane precedes every write to it.
    if (cluster > 1) {
      asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    } else {
      __syncthreads();
    }
    for (int i = threadIdx.x; i < n * W; i += kThreads) {
      const int4 at = places[i / W];
      if (at.x >= 0)
        *reinterpret_cast<int4*>(rows + at.z * p.stride_block + at.w * p.stride_offset + (i % W) * 16) = staging[i];
    }
    if (chunk == 0)
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const int4 at = places[i];
        if (at.x >= 0) scales[at.z * p.scale_block + at.w] = bytes[i];
      }
    __syncthreads();  // the staging is free for the next plane
  }
}

int staging_bytes(int per, int w) { return per * (w * 16 + kSlotBytes); }

template <int W>
int launch(const JtKvFp8CommitParams& p, int cluster, int sms, cudaStream_t stream) {
  const int chunks = p.head_dim / (16 * W);
  const int64_t planes = 2LL * p.num_layers * p.num_kv_heads * chunks;
  if (planes > 0x7fffffff) return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: too many planes");
  const int per = (p.num_slots + cluster - 1) / cluster;
  int rc = jt_cuda_check(cudaFuncSetAttribute(kv_fp8_commit_kernel<W>,
                                              cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemCap),
                         "kv_fp8_commit smem attribute");
  if (rc != JT_OK) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(planes, 16LL * sms) * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = staging_bytes(per, W);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return jt_cuda_check(cudaLaunchKernelEx(&cfg, kv_fp8_commit_kernel<W>, p, static_cast<int>(planes),
                                          chunks, per),
                       "kv_fp8_commit launch");
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

extern "C" int32_t jt_kv_fp8_commit_max_slots(void) {
  return kMaxSlots;
}

extern "C" int jt_kv_fp8_commit_launch(const JtKvFp8CommitParams* p, cudaStream_t stream) {
  if (p == nullptr) return jt_fail(JT_ERR_INVALID, "kv_fp8_commit: null params");
  if (p->num_slots < 0 || p->num_layers < 1 || p->num_kv_heads < 1 || p->head_dim < 16 ||
      p->head_dim % 16 != 0 || p->block_size < 1 || p->num_blocks < 1 || p->num_blocks > 0x7fffffff)
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
  // Whole 128-byte chunks (the widest that divide the row), by the smallest cluster whose CTAs
  // stage little enough to share an SM; the largest cluster may fill it.
  const int words = p->head_dim / 16;
  const int w = words % 8 == 0 ? 8 : words % 4 == 0 ? 4 : words % 2 == 0 ? 2 : 1;
  int cluster = 1;
  while (cluster < kMaxCluster && staging_bytes((p->num_slots + cluster - 1) / cluster, w) > kSmemShare)
    cluster *= 2;
  switch (w) {
    case 8: return launch<8>(*p, cluster, sms, stream);
    case 4: return launch<4>(*p, cluster, sms, stream);
    case 2: return launch<2>(*p, cluster, sms, stream);
    default: return launch<1>(*p, cluster, sms, stream);
  }
}
