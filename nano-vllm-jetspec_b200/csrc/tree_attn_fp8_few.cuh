// Attention over the 8-bit paged cache for requests of few query rows (nodes x query heads of a
// KV head <= 16: plain decode, chains of a few drafts).  Included by tree_attn_fp8.cu.
//
// Every byte of K and V is used by at most 16 rows, so the kernel is bound by HBM: per 128-key
// tile an SM has 1360 cycles at the measured copy rate, and all that matters is to spend fewer.
// It takes 1650: 16 requests of 30 to 32 thousand keys, 4 rows each, 183 us, 5.4 TB/s, and 184 to
// 198 by card with the merge and the launches (the 16-bit cache: 340).  The tensor core kernel needs
// 3400 (V expanded to bf16 through shared memory, 128-row MMAs with 4 live rows).  Launches whose
// node counts the host does not know (captured and compiled ones) take the form of 16 rows, 286 us
// for the same requests.  Here both products run as register mma.m16n8k16 on f16 with the keys (K)
// and the dims (V) on the 16 side and the query rows on the 8 side, so that up to 8 rows waste
// nothing, and the codes go from shared memory to MMA fragments in registers:
//   S^T = K Q^T   a lane holds 32 consecutive dims of keys g and g + 8 (g = lane / 4), two 16-byte
//                 loads a key, each 4-byte word the A fragment of one k-step after two exact
//                 e4m3x2 -> f16x2 conversions; Q's dims are permuted alike.
//   O^T = V^T P^T a lane holds dims 16 g .. 16 g + 15 of keys 2q, 2q+1, 2q+8, 2q+9 (q = lane % 4),
//                 one 16-byte load a key; byte permutes pair the keys.  P^T comes from S^T by
//                 movmatrix.
// Q enters as f16 after a power-of-two row scale (exact for bf16 but for elements 2^-22 below the
// row's largest).  2^e of the key multiplies its scores; 2^f of its value is folded into the
// exponent, y = x + f, P = 2^(y - M + 7) with M a lazy maximum of y (moved when exceeded by
// 2^8): P stays within 2^15, f16's range, and what f16 drops lies 2^-31 below the largest term.
// The sum has a lazy maximum m of its own, l = sum 2^(x - m): a key of small values may weigh
// most.  out = O / l 2^(M - 7 - m).  f16 and fp32 outputs add P's low parts (22 bits).
//
// Work: as in the tensor core kernel, the items' tiles form one line cut evenly over the SMs.
// Warp 0 loads (TMA, or cp.async rows where TMA cannot) through a ring of four 32 KB stages;
// each of the other warps takes 16 keys of a tile with its own maxima and sums, and the warps
// meet at the end of a piece.  Eight such warps (146 registers for up to 8 rows) beat sixteen of
// 96 (two tiles in hand) by 16 %.

constexpr int kFewStages = 4;
constexpr int kFewItemCost = 4;      // an item's fixed cost in tiles
constexpr int kFewMinPart = 5;
constexpr int kFewRowPitch = 136;    // floats per row of the meeting place

template <int NT>  // n-tiles of 8 rows
struct Few {
  static constexpr int kWarps = 8;                 // that take 16 keys of a tile each
  static constexpr int kThreads = 32 * (kWarps + 1);
  static constexpr int kRows = 8 * NT;
  static constexpr int kV = kFewStages * kTile8;
  static constexpr int kScale = 2 * kFewStages * kTile8;           // [stage][K, V][128] bytes
  static constexpr int kBad = kScale + kFewStages * 256;           // [stage][4] words: keys without a place
  static constexpr int kO = kBad + kFewStages * 16;                // [warp][row][pitch] float
  static constexpr int kMl = kO + kWarps * kRows * kFewRowPitch * 4;  // [warp][row] m, l, M, -
  static constexpr int kMisc = kMl + kWarps * kRows * 16;          // scan; abort
  static constexpr int kBar = kMisc + 512;
  static constexpr int kBytes = kBar + 8 * 2 * kFewStages + 1024;
  static_assert(kBytes <= 227 * 1024, "shared memory per CTA");
};

__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return h;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) { return jt::MmaOp<__half>::pack(lo, hi); }
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// A NaN code of a key that some row does not see must not reach that row as 0 x NaN: V's come out
// as 448 in the tiles that hold such keys, and note_nan_codes sees to the rows that do see it.
__device__ __forceinline__ uint32_t finite_f16x2(uint32_t v) {
  uint32_t r;
  asm("min.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(v), "r"(0x5f005f00u));  // 448
  return r;
}

__device__ __noinline__ void note_nan_keys(const JtTreeAttnFp8Params& p, uint4 a, uint4 b, uint4 c, uint4 d) {
  if ((nan_codes(a) | nan_codes(b) | nan_codes(c) | nan_codes(d)) != 0) note_nan_codes(p);
}

struct FewPiece {
  int r, h, P, T, q_start, t0, n, key_end, slot, finishes;
};
// Walks this CTA's part of the line; every warp keeps its own.
struct FewCursor {
  int64_t x0, x1, s_item;
  int r, h, P, T;
  bool more;
};
__device__ __forceinline__ int2 few_request(const JtTreeAttnFp8Params& p, int r, bool flag, int most) {
  int2 q = load_request(p, r, flag);
  if (q.y * p.groups > most) q.y = 0;  // the other kernel's, or clear_refused
  return q;
}
__device__ __forceinline__ int few_cost(int P, int T) {
  return T == 0 ? 0 : ((P + T + kN - 1) >> 7) + kFewItemCost;
}
__device__ __noinline__ bool few_next(const JtTreeAttnFp8Params& p, FewCursor& c, FewPiece& it, int most) {
  while (c.more) {
    const int n = (c.P + c.T + kN - 1) >> 7;
    const ItemInfo info{c.P + c.T, n, 0, 1, n + kFewItemCost};
    const int tb = cut_tile(info, c.s_item, c.x0), te = cut_tile(info, c.s_item, c.x1);
    const bool found = te > tb;
    if (found) {
      it.r = c.r; it.h = c.h; it.P = c.P; it.T = c.T;
      it.q_start = __ldg(p.cu_seqlens_q + c.r);
      it.t0 = tb; it.n = te - tb; it.key_end = c.P + c.T;
      it.finishes = te == n;
      it.slot = tb == 0 && te == n ? -1 : 2 * static_cast<int>(blockIdx.x) + (tb == 0 ? 1 : 0);
    }
    c.s_item += info.cost;
    if (c.s_item >= c.x1) {
      c.more = false;
    } else if (++c.h == p.num_kv_heads) {
      c.h = 0;
      c.T = 0;
      while (c.T == 0 && ++c.r < p.num_requests) {
        const int2 q = few_request(p, c.r, false, most);
        c.P = q.x;
        c.T = q.y;
      }
      if (c.r >= p.num_requests) c.more = false;
    }
    if (found) return true;
  }
  return false;
}

template <int NT, bool kWide, typename QT>
__global__ void __launch_bounds__(Few<NT>::kThreads, 1)
    tree_attn_fp8_few_kernel(const __grid_constant__ JtTreeAttnFp8Params p,
                             const __grid_constant__ CUtensorMap kmap,
                             const __grid_constant__ CUtensorMap vmap, const LoadPlan plan) {
  using F = Few<NT>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = jt::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* sbase = smem_raw + (base - raw);
  const uint32_t full0 = base + F::kBar, empty0 = full0 + 8 * kFewStages;
  int64_t* scan = reinterpret_cast<int64_t*>(sbase + F::kMisc);
  volatile int* abort = reinterpret_cast<volatile int*>(sbase + F::kMisc + 504);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (tid == 0) *abort = 0;
  if (tid < 2 * kFewStages) {
    // Full: every lane of the loading warp twice (rows by cp.async and their scale bytes, or
    // TMA).  Empty: the eight warps of the tile.
    mbar_init(full0 + 8 * tid, tid < kFewStages ? 64 : 8);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_proxy_async();
  }
  // This CTA's part of the line, as in the tensor core kernel.
  const int R = p.num_requests, per = (R + F::kThreads - 1) / F::kThreads;
  const int r_lo = min(tid * per, R), r_hi = min(r_lo + per, R);
  int64_t mine = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    const int2 q = few_request(p, r, blockIdx.x == 0, F::kRows);
    mine += static_cast<int64_t>(few_cost(q.x, q.y)) * p.num_kv_heads;
  }
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t before = 0, total = 0;
  for (int k = 0; k <= F::kWarps; ++k) {
    if (k < warp) before += scan[k];
    total += scan[k];
  }
  const int64_t my_start = before + incl - mine;
  const int parts = static_cast<int>(
      max(static_cast<int64_t>(1), min(static_cast<int64_t>(gridDim.x), total / kFewMinPart)));
  const bool has_part = static_cast<int>(blockIdx.x) < parts && total > 0;
  FewCursor cur{};
  cur.x0 = has_part ? total * blockIdx.x / parts : 0;
  cur.x1 = has_part ? total * (blockIdx.x + 1) / parts : 0;
  if (has_part && mine > 0 && my_start <= cur.x0 && cur.x0 < my_start + mine) {
    int64_t s = my_start;
    for (int r = r_lo; r < r_hi; ++r) {
      const int2 q = few_request(p, r, false, F::kRows);
      const int64_t c = static_cast<int64_t>(few_cost(q.x, q.y)) * p.num_kv_heads;
      if (cur.x0 < s + c) {
        scan[32] = r;
        scan[33] = s;
        break;
      }
      s += c;
    }
  }
  __syncthreads();
  cur.more = has_part;
  if (has_part) {
    cur.r = static_cast<int>(scan[32]);
    const int2 q = few_request(p, cur.r, false, F::kRows);
    cur.P = q.x;
    cur.T = q.y;
    const int64_t s = scan[33], c = few_cost(q.x, q.y);
    cur.h = static_cast<int>((cur.x0 - s) / c);
    cur.s_item = s + c * cur.h;
  }

  FewPiece it;
  uint32_t g0 = 0;  // tiles of earlier pieces
  if (warp == 0) {
    // ------------------------------------------------------------------ loads
    int meta_valid[2] = {0, 0};
    PieceMeta* meta = carve(p.workspace).meta + 2 * blockIdx.x;
    const char* kp = static_cast<const char*>(p.k_pool);
    const char* vp = static_cast<const char*>(p.v_pool);
    const unsigned char* ksc = static_cast<const unsigned char*>(p.k_scale);
    const unsigned char* vsc = static_cast<const unsigned char*>(p.v_scale);
    const int chunks = p.head_dim / 16, boxes = plan.tma ? kN / plan.box : 1;
    if (lane == 0) meta[0].nan = meta[1].nan = 0;  // before any tile: note_nan_codes
    bool dead = false, gathered = false;
    uint32_t issued = 0, marked = ~0u;  // stages whose words of missing keys may not be zero
#pragma unroll 1
    while (!dead && few_next(p, cur, it, F::kRows)) {
      if (it.slot >= 0) {
        const int which = it.slot & 1;
        meta_valid[which] = 1;
        if (lane == 0) {
          meta[which].finishes = it.finishes;
          meta[which].r = it.r;
          meta[which].h = it.h;
          meta[which].mb = 0;
        }
      }
      const int32_t* table = p.block_tables + static_cast<int64_t>(it.r) * p.table_stride0;
      int batch = -1, pages = -1;  // a lane's box of 32 consecutive ones, looked up together
      uint32_t lost = 0;           // those of them whose page lies outside the pool
#pragma unroll 1
      for (int t = 0; t < it.n; ++t) {
        const uint32_t g = g0 + t, stage = g % kFewStages;
        const int tile = it.t0 + t, kb = tile * kN;
        const uint32_t full = full0 + 8 * stage;
        const uint32_t kdst = base + stage * kTile8, vdst = kdst + F::kV;
        unsigned char* sc = sbase + F::kScale + stage * 256;
        uint32_t* none = reinterpret_cast<uint32_t*>(sbase + F::kBad) + 4 * stage;
        const bool tma = plan.tma && kb + kN <= it.P;
        if (tma && (tile * boxes) >> 5 != batch) {
          batch = (tile * boxes) >> 5;
          const int pos = (32 * batch + lane) * plan.box;
          pages = pos < it.P ? __ldg(table + pos / p.block_size) : -1;
          const bool bad = pos < it.P && (pages < 0 || pages >= p.num_blocks);
          if (bad) {
            atomicOr(&g_attn_fp8_errors, JT_DEVERR_OUT_OF_RANGE);
            pages = -1;
          }
          lost = __ballot_sync(0xffffffffu, bad);
        }
        KeyPlace at[4];
        if (!tma) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            at[i] = locate_key(p, table, kb + 32 * i + lane, it.P, it.key_end, it.q_start);
        }
        if (g >= kFewStages)
          mbar_wait(empty0 + 8 * stage, ((g / kFewStages) & 1) ^ 1, abort);
        dead = __shfl_sync(0xffffffffu, *abort, 0) != 0;
        if (dead) break;
        issued = g + 1;
        if (tma) {
          if (gathered) fence_proxy_async();
          if (lane == 0) mbar_arrive_tx(full, 2 * kTile8 + 2 * kN);
          __syncwarp();
          const int page = __shfl_sync(0xffffffffu, pages, (tile * boxes + lane) & 31);
          if (lane < boxes) {
            // Page -1 lies outside the map: zeros.
            const int i = lane * plan.box, off = (kb + i) % p.block_size;
            tma_load_4d(kdst + i * kD, &kmap, 0, it.h, off, page, full);
            tma_load_4d(vdst + i * kD, &vmap, 0, it.h, off, page, full);
            const int64_t pg = max(page, 0);
            const uint32_t sdst = base + F::kScale + stage * 256 + i;
            bulk_load(sdst, ksc + pg * p.ks_stride0 + it.h * p.ks_stride1 + off, plan.box, full);
            bulk_load(sdst + kN, vsc + pg * p.vs_stride0 + it.h * p.vs_stride1 + off, plan.box, full);
          }
          if (lost != 0 || (marked >> stage) & 1u) {
            if (lane < 4) {
              // This word's 32 keys lie in one box, or in two of 16.
              const uint32_t b = lost >> (((tile * boxes) & 31) + 32 * lane / plan.box);
              none[lane] = plan.box >= 32 ? (b & 1u ? ~0u : 0u) : (b & 1u ? 0xffffu : 0u) | (b & 2u ? ~0xffffu : 0u);
            }
            marked = (marked & ~(1u << stage)) | (lost != 0 ? 1u << stage : 0u);
          }
          if (lane != 0) mbar_arrive(full);
          mbar_arrive(full);
        } else {
          gathered = true;
          marked |= 1u << stage;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool ok = at[i].page >= 0;
            const int64_t page = ok ? at[i].page : 0;
            const int off = at[i].off, row = 32 * i + lane;
            gather_row(kdst, row, kp + page * p.k_stride0 + off * p.k_stride1 + it.h * p.k_stride2, ok ? chunks : 0);
            gather_row(vdst, row, vp + page * p.v_stride0 + off * p.v_stride1 + it.h * p.v_stride2, ok ? chunks : 0);
            sc[row] = ok ? __ldg(ksc + page * p.ks_stride0 + it.h * p.ks_stride1 + off) : 127;
            sc[kN + row] = ok ? __ldg(vsc + page * p.vs_stride0 + it.h * p.vs_stride1 + off) : 127;
            const uint32_t out = __ballot_sync(0xffffffffu, !ok);
            if (lane == 0) none[i] = out;
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(full) : "memory");
          mbar_arrive(full);
        }
      }
      g0 += it.n;
    }
    // The copies of the last stages have landed before the CTA exits.
    asm volatile("cp.async.wait_all;\n" ::: "memory");
    for (uint32_t g = issued > kFewStages ? issued - kFewStages : 0; g < issued; ++g)
      mbar_wait(full0 + 8 * (g % kFewStages), (g / kFewStages) & 1, abort, false);
    if (lane == 0) {
      meta[0].valid = meta_valid[0];
      meta[1].valid = meta_valid[1];
    }
    return;
  }

  // -------------------------------------------------------------------- keys
  const int w = warp - 1;
  const int g8 = lane >> 2, q4 = lane & 3;
  const float log2e = 1.4426950408889634f;
  float* o_place = reinterpret_cast<float*>(sbase + F::kO);
  float4* ml_place = reinterpret_cast<float4*>(sbase + F::kMl);
#pragma unroll 1
  while (few_next(p, cur, it, F::kRows)) {  // to the end even after a wait that ran out: the warps meet
    const int rows = it.T * p.groups;
    // Q fragments: row g8 of each n-tile, dims 32 q4 .. 32 q4 + 31, as f16 of row / 2^e.
    uint32_t qf[NT][16];
    float c_row[NT][2];  // factors of rows 2 q4 and 2 q4 + 1
    uint32_t seen[NT][2];  // tree nodes those rows see
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int row = 8 * t + g8, node = row / p.groups;
      const QT* src = static_cast<const QT*>(p.q) + (static_cast<int64_t>(it.q_start) + node) * p.q_stride0 +
                      (static_cast<int64_t>(it.h) * p.groups + row - node * p.groups) * p.q_stride1 + 32 * q4;
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows && 32 * q4 + 8 * i < p.head_dim) v = __ldg(reinterpret_cast<const uint4*>(src) + i);
        qf[t][4 * i] = v.x;
        qf[t][4 * i + 1] = v.y;
        qf[t][4 * i + 2] = v.z;
        qf[t][4 * i + 3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = __vmaxu2(top, qf[t][i] & 0x7fff7fffu);
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = __float_as_uint(jt::MmaOp<QT>::unpack(max(top & 0xffffu, top >> 16)).x);
      const bool finite = top < 0x7f800000u;
      const int e = top != 0 && finite ? max(static_cast<int>(top >> 23) - 134, -126) : 0;  // to [2^7, 2^8)
      const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 x = jt::MmaOp<QT>::unpack(qf[t][i]);
        qf[t][i] = pack_f16(x.x * inv, x.y * inv);
      }
      // A row with a non-finite element: its factor makes its scores NaN.
      const float c = finite ? p.scale * log2e * __uint_as_float(static_cast<uint32_t>(127 + e) << 23)
                             : __uint_as_float(0x7fc00000u);
      c_row[t][0] = __shfl_sync(0xffffffffu, c, 8 * q4);
      c_row[t][1] = __shfl_sync(0xffffffffu, c, 8 * q4 + 4);
      seen[t][0] = seen[t][1] = 0;
    }
    if ((it.t0 + it.n) * kN > it.P) {
      // Visibility bits: lane n reads the bias of node n, a ballot collects a node's word.
      const float* bias = p.qq_bias + __ldg(p.qq_bias_offsets + it.r);
#pragma unroll 4
      for (int j = 0; j < it.T; ++j) {
        const uint32_t word = __ballot_sync(0xffffffffu, lane <= j && __ldg(bias + j * it.T + min(lane, j)) == 0.f);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if ((8 * t + 2 * q4 + i) / p.groups == j) seen[t][i] = word;
      }
    }
    float o[NT][8][4];
    float m[NT][2], l[NT][2], my[NT][2];  // of x, of y
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = my[t][0] = my[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][j][i] = 0.f;
    }
#pragma unroll 1
    for (int t = 0; t < it.n; ++t) {
      const uint32_t g = g0 + t, stage = g % kFewStages;
      const int key0 = (it.t0 + t) * kN + 16 * w;
      mbar_wait(full0 + 8 * stage, (g / kFewStages) & 1, abort);
      __syncwarp();
      const unsigned char* kt = sbase + stage * kTile8 + 16 * w * 128;
      const unsigned char* vt = kt + F::kV;
      const unsigned char* sc = sbase + F::kScale + stage * 256 + 16 * w;
      // Keys without a place in the pool are left out, like tree nodes that a row does not see.
      const uint32_t none = (reinterpret_cast<const uint32_t*>(sbase + F::kBad)[4 * stage + (w >> 1)] >>
                             (16 * (w & 1))) & 0xffffu;
      const bool tail = (it.t0 + t + 1) * kN > it.P, masked = tail || none != 0;
      // S^T
      float s[NT][2][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][0][i] = s[n][1][i] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int off = g8 * 128 + (((2 * q4 + c) ^ (g8 & 7)) << 4);
        const uint4 a = *reinterpret_cast<const uint4*>(kt + off);
        const uint4 b = *reinterpret_cast<const uint4*>(kt + 1024 + off);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t a0 = e4m3x2_f16x2(aw[i]), a1 = e4m3x2_f16x2(bw[i]);
          const uint32_t a2 = e4m3x2_f16x2(aw[i] >> 16), a3 = e4m3x2_f16x2(bw[i] >> 16);
          const int k = 4 * c + i;
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_f16(s[n][i & 1], a0, a1, a2, a3, qf[n][2 * k], qf[n][2 * k + 1]);
        }
      }
      // V of this lane's four keys, before the stage is given back.
      uint4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = 2 * q4 + (i & 1) + 8 * (i >> 1);
        v[i] = *reinterpret_cast<const uint4*>(vt + key * 128 + ((g8 ^ (key & 7)) << 4));
      }
      if (tail) note_nan_keys(p, v[0], v[1], v[2], v[3]);
      const uint32_t kb0 = sc[g8], kb1 = sc[g8 + 8], vb0 = sc[kN + g8], vb1 = sc[kN + g8 + 8];
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * stage);
      // A NaN value row makes the scores of its key NaN for the rows that see it.
      const float kf[2] = {scale_value(vb0 == 255u ? 255u : kb0), scale_value(vb1 == 255u ? 255u : kb1)};
      const float fe[2] = {static_cast<float>(static_cast<int>(vb0) - 127), static_cast<float>(static_cast<int>(vb1) - 127)};
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float x[2][2];  // [key g8, g8 + 8][row 2 q4, 2 q4 + 1]
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            x[k][i] = (s[n][0][2 * k + i] + s[n][1][2 * k + i]) * kf[k] * c_row[n][i];
        if (masked) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int node = key0 + g8 + 8 * k - it.P;
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if ((none >> (g8 + 8 * k)) & 1u || (node >= 0 && !(node < 16 && (seen[n][i] >> node) & 1u)))
                x[k][i] = -INFINITY;
          }
        }
        bool moves = false;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          moves |= fmaxf(x[0][i], x[1][i]) > m[n][i] + 8.f ||
                   fmaxf(x[0][i] + fe[0], x[1][i] + fe[1]) > my[n][i] + 8.f;
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(x[0][i], x[1][i]), topy = fmaxf(x[0][i] + fe[0], x[1][i] + fe[1]);
#pragma unroll
            for (int d = 4; d < 32; d *= 2) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
              topy = fmaxf(topy, __shfl_xor_sync(0xffffffffu, topy, d));
            }
            if (top > m[n][i] + 8.f) {
              if (m[n][i] != -INFINITY) l[n][i] *= jt::fast_exp2(m[n][i] - top);
              m[n][i] = top;
            }
            if (topy > my[n][i] + 8.f) {
              const float alpha = my[n][i] == -INFINITY ? 1.f : jt::fast_exp2(my[n][i] - topy);
              my[n][i] = topy;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                o[n][j][i] *= alpha;
                o[n][j][2 + i] *= alpha;
              }
            }
          }
        }
        float e[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float nm = m[n][i] == -INFINITY ? 0.f : -m[n][i];
          const float ny = my[n][i] == -INFINITY ? 0.f : 7.f - my[n][i];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            e[k][i] = jt::fast_exp2(x[k][i] + (fe[k] + ny));
            l[n][i] += jt::fast_exp2(x[k][i] + nm);
          }
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t hi = pack_f16(e[k][0], e[k][1]);
          ph[n][k] = transpose8(hi);
          if constexpr (kWide) {
            const float2 f = jt::MmaOp<__half>::unpack(hi);
            pl[n][k] = transpose8(pack_f16(e[k][0] - f.x, e[k][1] - f.y));
          }
        }
      }
      // O^T
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t vw[4] = {i == 0 ? v[0].x : i == 1 ? v[0].y : i == 2 ? v[0].z : v[0].w,
                                i == 0 ? v[1].x : i == 1 ? v[1].y : i == 2 ? v[1].z : v[1].w,
                                i == 0 ? v[2].x : i == 1 ? v[2].y : i == 2 ? v[2].z : v[2].w,
                                i == 0 ? v[3].x : i == 1 ? v[3].y : i == 2 ? v[3].z : v[3].w};
#pragma unroll
        for (int k = 0; k < 2; ++k) {  // dims 16 g8 + 4 i + 2 k, + 1
          const uint32_t sel = k ? 0x7362u : 0x5140u;
          const uint32_t ab = __byte_perm(vw[0], vw[1], sel), cd = __byte_perm(vw[2], vw[3], sel);
          uint32_t a0 = e4m3x2_f16x2(ab), a1 = e4m3x2_f16x2(ab >> 16);
          uint32_t a2 = e4m3x2_f16x2(cd), a3 = e4m3x2_f16x2(cd >> 16);
          if (tail) {
            a0 = finite_f16x2(a0);
            a1 = finite_f16x2(a1);
            a2 = finite_f16x2(a2);
            a3 = finite_f16x2(a3);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(o[n][2 * i + k], a0, a1, a2, a3, ph[n][0], ph[n][1]);
            if constexpr (kWide) mma_f16(o[n][2 * i + k], a0, a1, a2, a3, pl[n][0], pl[n][1]);
          }
        }
      }
    }
    g0 += it.n;
    // The warps meet: every one leaves its maxima, sums and O, a thread joins four dims of a row.
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * F::kWarps) : "memory");  // the place is free
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[n][i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int row = 8 * n + 2 * q4 + i;
        if (g8 == 0) ml_place[w * F::kRows + row] = make_float4(m[n][i], sum, my[n][i], 0.f);
        float2* dst = reinterpret_cast<float2*>(o_place + (w * F::kRows + row) * kFewRowPitch + 16 * g8);
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[j] = make_float2(o[n][j][i], o[n][j][2 + i]);
      }
    asm volatile("bar.sync 1, %0;\n" ::"n"(32 * F::kWarps) : "memory");
    const int row = (tid - 32) >> 5, d = 4 * lane;  // a warp a row
    for (int rw = row; rw < rows; rw += F::kWarps) {
      float top = -INFINITY, topy = -INFINITY;
#pragma unroll
      for (int k = 0; k < F::kWarps; ++k) {
        top = fmaxf(top, ml_place[k * F::kRows + rw].x);
        topy = fmaxf(topy, ml_place[k * F::kRows + rw].z);
      }
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < F::kWarps; ++k) {
        const float4 a = ml_place[k * F::kRows + rw];
        // Keys without a maximum have zero sums, or NaN ones that have to stay.
        const float f = a.z == -INFINITY ? 1.f : jt::fast_exp2(a.z - topy);
        const float4 x = *reinterpret_cast<const float4*>(o_place + (k * F::kRows + rw) * kFewRowPitch + d);
        sum = fmaf(a.y, a.x == -INFINITY ? 1.f : jt::fast_exp2(a.x - top), sum);
        acc = make_float4(fmaf(x.x, f, acc.x), fmaf(x.y, f, acc.y), fmaf(x.z, f, acc.z), fmaf(x.w, f, acc.w));
      }
      const Workspace ws = carve(p.workspace);
      if (it.slot >= 0) {
        if (lane == 0) {
          ws.ml[it.slot * 2ll * kM + rw] = make_float2(top, sum);
          ws.ml[(it.slot * 2ll + 1) * kM + rw] = make_float2(topy, 0.f);
        }
        ws.o[(it.slot * 2ll * kM + rw) * (kD / 4) + lane] = acc;
      } else if (d < p.head_dim) {
        store_row4<kWide>(p, it.q_start, it.h, rw, d, acc, sum, topy - 7.f - top);
      }
    }
  }
}

// Merge of items cut between CTAs: block c takes the item that begins in CTA c's part and ends in
// a later one, a warp per row.
template <bool kWide>
__global__ void __launch_bounds__(32 * kFewRows) tree_attn_fp8_few_merge_kernel(
    const __grid_constant__ JtTreeAttnFp8Params p, const int parts, const int most) {
  // With no kernel after it for the requests that this one does not take.
  if (most > 0 && threadIdx.x < 32) clear_refused(p, 1, most);
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const Workspace w = carve(p.workspace);
  const int c = blockIdx.x, row = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PieceMeta first = w.meta[2 * c + 1];
  if (first.nan != 0) spread_nan_codes(p, 1, kFewRows);
  if (!first.valid || first.finishes) return;
  if (row >= p.node_counts[first.r] * p.groups) return;
  int nan = 0;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, my = -INFINITY, l = 0.f;
  for (int i = c; i < parts; ++i) {
    const int slot = i == c ? 2 * c + 1 : 2 * i;
    if (i != c && !w.meta[slot].valid) continue;  // a part shorter than the least cut
    nan |= w.meta[slot].nan;
    const float2 ml = w.ml[slot * 2ll * kM + row];
    const float oy = w.ml[(slot * 2ll + 1) * kM + row].x;
    const float4 o = w.o[(slot * 2ll * kM + row) * (kD / 4) + lane];
    // A row whose keys were all NaN has no maximum but NaN sums, which have to stay.
    auto factor = [](float own, float top) { return own == -INFINITY ? 1.f : jt::fast_exp2(own - top); };
    const float top = fmaxf(m, ml.x), topy = fmaxf(my, oy);
    const float fa = factor(my, topy), fb = factor(oy, topy);
    l = l * factor(m, top) + ml.y * factor(ml.x, top);
    acc = make_float4(acc.x * fa + o.x * fb, acc.y * fa + o.y * fb, acc.z * fa + o.z * fb, acc.w * fa + o.w * fb);
    m = top;
    my = topy;
    if (i != c && w.meta[slot].finishes) break;
  }
  if (nan != 0 && sees_nan_code(p, first.r, load_request(p, first.r, false), first.h, row / p.groups))
    l = __uint_as_float(0x7fc00000u);
  if (4 * lane < p.head_dim)
    store_row4<kWide>(p, p.cu_seqlens_q[first.r], first.h, row, 4 * lane, acc, l, my - 7.f - m);
}

template <int NT, bool kWide, typename QT>
int launch_few(const JtTreeAttnFp8Params& p, const LoadPlan& plan, const CUtensorMap& kmap,
               const CUtensorMap& vmap, int grid, bool alone, cudaStream_t stream) {
  auto kernel = tree_attn_fp8_few_kernel<NT, kWide, QT>;
  int rc = jt_cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              Few<NT>::kBytes),
                         "tree_attn_fp8 smem attribute");
  if (rc != JT_OK) return rc;
  kernel<<<grid, Few<NT>::kThreads, Few<NT>::kBytes, stream>>>(p, kmap, vmap, plan);
  rc = jt_cuda_check(cudaGetLastError(), "tree_attn_fp8 few rows launch");
  if (rc != JT_OK) return rc;
  return launch_dependent(tree_attn_fp8_few_merge_kernel<kWide>, dim3(grid), 32 * kFewRows, 0, stream,
                          "tree_attn_fp8 few rows merge launch", p, grid, alone ? Few<NT>::kRows : 0);
}
