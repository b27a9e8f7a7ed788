// Block tables, slot maps and positions of a round, built on the GPU from request lengths.
//
// For request r with c = cached_lens[r] tokens in the cache and n = new_lens[r] to write:
//   have = ceil(c / B), need = ceil((c + n) / B)         pages before and after (B = block_size)
//   first(r) = sum over earlier requests of need - have  its first entry of the free list
//   block_tables[r, have + i] = free_pages[first(r) + i]     i < need - have
//   token t of r: position p = c + t, slot = page(p / B) * B + p % B
// Every CTA scans all the requests' lengths itself (integer adds: the same result in each),
// so one launch with no grid-wide dependency does the whole round; a token's page that this
// round takes is read from the free list, not from the table entry another CTA writes.
//
// Bound: a launch and a few dependent loads for a decode round (R lengths, one scan, one
// token each); 20 written bytes per token for a prefill round.  One thread per request up to
// kThreads requests, contiguous runs of requests per thread above; tokens and pages then
// find their request by binary search over the threads' offsets in shared memory.
#include <algorithm>

#include "common.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kTokensPerCta = 2 * kThreads;

__device__ uint32_t g_maps_errors;

// Lengths of one request: tokens, and the pages it takes from the free list.
struct Lens {
  int cached, fresh, have, take;
};
__device__ __forceinline__ Lens load_lens(const JtRequestMapsParams& p, int r) {
  Lens l;
  l.cached = max(__ldg(p.cached_lens + r), 0);
  l.fresh = max(__ldg(p.new_lens + r), 0);
  const int b = p.block_size;
  l.have = l.cached / b + (l.cached % b != 0);
  const int64_t end = static_cast<int64_t>(l.cached) + l.fresh;
  l.take = static_cast<int>((end + b - 1) / b) - l.have;
  return l;
}

// Last index i in [0, kThreads) with offsets[i] <= x (offsets ascending, offsets[0] = 0).
__device__ __forceinline__ int owner(const int64_t* offsets, int64_t x) {
  int lo = 0;
#pragma unroll
  for (int step = kThreads / 2; step > 0; step >>= 1)
    if (offsets[lo + step] <= x) lo += step;
  return lo;
}

__global__ void __launch_bounds__(kThreads) request_maps_kernel(const JtRequestMapsParams p) {
  __shared__ int64_t tok_off[kThreads], page_off[kThreads];  // before each thread's requests
  __shared__ int64_t warp_tok[kThreads / 32], warp_page[kThreads / 32];
  __shared__ int64_t total_tok, total_page;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int R = p.num_requests, B = p.block_size;
  const int per = (R + kThreads - 1) / kThreads;
  const int r0 = min(tid * per, R), r1 = min(r0 + per, R);

  int64_t tok = 0, pages = 0;
  bool bad = false;
  for (int r = r0; r < r1; ++r) {
    const Lens l = load_lens(p, r);
    bad |= __ldg(p.cached_lens + r) < 0 || __ldg(p.new_lens + r) < 0;
    tok += l.fresh;
    pages += l.take;
  }
  int64_t a = tok, b = pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t ya = __shfl_up_sync(0xffffffffu, a, o);
    const int64_t yb = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += ya; b += yb; }
  }
  if (lane == 31) { warp_tok[warp] = a; warp_page[warp] = b; }
  __syncthreads();
  int64_t base_t = 0, base_p = 0;
  for (int k = 0; k < warp; ++k) { base_t += warp_tok[k]; base_p += warp_page[k]; }
  const int64_t my_tok = base_t + a - tok, my_page = base_p + b - pages;
  tok_off[tid] = my_tok;
  page_off[tid] = my_page;
  if (tid == kThreads - 1) { total_tok = base_t + a; total_page = base_p + b; }
  __syncthreads();

  // Per-request outputs: each CTA writes a share of the threads' runs.
  if (tid % gridDim.x == blockIdx.x) {
    int64_t run = my_tok;
    for (int r = r0; r < r1; ++r) {
      const Lens l = load_lens(p, r);
      p.cu_seqlens[r] = static_cast<int32_t>(run);
      p.context_lens[r] = l.cached + l.fresh;
      run += l.fresh;
    }
    if (bad) atomicOr(&g_maps_errors, JT_DEVERR_OUT_OF_RANGE);
  }
  if (blockIdx.x == 0 && tid == 0) {
    p.cu_seqlens[R] = static_cast<int32_t>(total_tok);
    p.pages_taken[0] = static_cast<int32_t>(total_page);
  }

  // New table entries, one per taken page.  A free list that is too short gives -1.
  const int64_t grid_threads = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  for (int64_t i = first; i < total_page; i += grid_threads) {
    const int t = owner(page_off, i);
    int64_t run = page_off[t];
    for (int r = t * per;; ++r) {
      const Lens l = load_lens(p, r);
      if (i < run + l.take) {
        const int64_t col = l.have + (i - run);
        if (col < p.table_width)
          p.block_tables[r * p.table_stride0 + col] = i < p.num_free ? __ldg(p.free_pages + i) : -1;
        break;
      }
      run += l.take;
    }
  }

  // Tokens; entries past the round's total are padding that the cache writes skip.
  for (int64_t i = first; i < p.max_tokens; i += grid_threads) {
    int64_t slot = -1, position = 0;
    int request = -1;
    if (i < total_tok) {
      const int t = owner(tok_off, i);
      int64_t run_t = tok_off[t], run_p = page_off[t];
      for (int r = t * per;; ++r) {
        const Lens l = load_lens(p, r);
        if (i < run_t + l.fresh) {
          const int pos = l.cached + static_cast<int>(i - run_t);
          const int col = pos / B;
          int page = -1;
          if (col < p.table_width) {
            if (col < l.have) {
              page = p.block_tables[r * p.table_stride0 + col];
            } else {
              const int64_t f = run_p + (col - l.have);
              if (f < p.num_free) page = __ldg(p.free_pages + f);
            }
          }
          if (page >= 0) slot = static_cast<int64_t>(page) * B + (pos - col * B);
          position = pos;
          request = r;
          break;
        }
        run_t += l.fresh;
        run_p += l.take;
      }
    }
    p.slot_mapping[i] = slot;
    p.positions[i] = position;
    p.token_to_request[i] = request;
  }
}

}  // namespace

int jt_read_errors_maps(uint32_t* bits) {
  uint32_t zero = 0;
  int rc = jt_cuda_check(cudaMemcpyFromSymbol(bits, g_maps_errors, sizeof(uint32_t)),
                         "read request-map error word");
  if (rc != JT_OK) return rc;
  return jt_cuda_check(cudaMemcpyToSymbol(g_maps_errors, &zero, sizeof(uint32_t)),
                       "clear request-map error word");
}

extern "C" int jt_request_maps_launch(const JtRequestMapsParams* p, cudaStream_t stream) {
  if (p == nullptr) return jt_fail(JT_ERR_INVALID, "request_maps: null params");
  if (p->num_requests < 1 || p->block_size < 1 || p->table_width < 1 || p->num_free < 0 ||
      p->max_tokens < 0 || p->table_stride0 < p->table_width)
    return jt_fail(JT_ERR_INVALID, "request_maps: invalid geometry");
  if (!p->block_tables || !p->cached_lens || !p->new_lens || (p->num_free > 0 && !p->free_pages) ||
      !p->cu_seqlens || !p->context_lens || !p->pages_taken ||
      (p->max_tokens > 0 && (!p->slot_mapping || !p->positions || !p->token_to_request)))
    return jt_fail(JT_ERR_INVALID, "request_maps: null tensor pointer");
  int dev = 0, sms = 0;
  int rc = jt_cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc != JT_OK) return rc;
  rc = jt_cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev),
                     "SM count");
  if (rc != JT_OK) return rc;
  const int64_t want = (static_cast<int64_t>(p->max_tokens) + kTokensPerCta - 1) / kTokensPerCta;
  const int grid = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, 2LL * sms)));
  request_maps_kernel<<<grid, kThreads, 0, stream>>>(*p);
  return jt_cuda_check(cudaGetLastError(), "request_maps launch");
}
