// Packed tree attention over an 8-bit paged cache (e4m3 codes, power-of-two row scales) on
// tcgen05 tensor cores.
//
// For query row i (node j, head hq) of request r: keys are positions 0..P+T-1 (prefix pages,
// then the T tree nodes), visible when the position is below P, or is node n <= j with zero
// bias.  With k = K 2^e, v = V 2^f (K, V codes):
//   s = scale * 2^e * sum_d q_d K_d,   p = exp(s - max),   out = sum p 2^f V / sum p
// * Scores on 8-bit operands: a bf16 query element, scaled by the row's power of two, is the sum
//   of two e4m3 values (4 significant bits each, the second one signed: 8 bits), an f16 one of
//   three.  Q enters as two or three e4m3 tiles against the same K tile (kind::f8f6f4 runs at
//   twice the bf16 rate, so two terms cost what one bf16 product would), and K goes from HBM to
//   the tensor core untouched.  2^e multiplies the score column in the softmax.  Exact but for
//   elements below 2^-9.8 (f16: 2^-6.8) of the row's largest: with that one scaled into
//   (224, 448] the terms end at e4m3's least spacing 2^-9, so they lose at most half of it,
//   2^-10 / 224 = 2^-17.8 of the largest.
// * PV runs in bf16: four warps expand the V codes (exact in bf16, 2^f folded in) into the
//   swizzled tile the MMA reads.  P is rounded to bf16 (8 bits, as in the 16-bit cache's
//   kernel); f16 and fp32 outputs take P as hi + lo bf16 (16 bits).
//
// Requests of up to 16 rows (nodes x query heads of a KV head) would leave seven eighths of a
// 128-row tile empty and take the kernel of tree_attn_fp8_few.cuh.  In one process 16 requests of
// 30 to 32 thousand keys take 210 us there and 401 here with 4 rows each, 282 and 404 with 16, and
// 64 requests of 500 to 4000 keys 115 and 160 with 4 rows, 156 and 164 with 16.
//
// Work: an item is (request, KV head, m-block), an m-block one or two 128-row query tiles;
// the items' 128-key tiles, weighted by their measured time, form one line that is cut into
// equal parts, one per CTA, so every SM has the same to do whatever the lengths (weights of 1
// and 2 for one and two query tiles and 3 for an item, by tensor time alone, left CTAs between
// 411 and 735 us of the same mix).  Every CTA scans the lengths itself and finds its part: no plan
// kernel, no queue.  An item cut between CTAs leaves unnormalised fp32 partials that a second small
// kernel merges (a programmatic dependent, which also writes the rows of refused requests and of
// NaN codes).
//
// Two softmax streams per CTA keep the tensor core busy while the other one works.  With two
// query tiles (trees of more than 128 rows) each stream owns a tile and both use every K / V
// tile; with one, each takes half of every key tile and their (max, sum, O) are merged at the
// end.  A stream goes through its keys 64 at a time, in two score buffers with a warpgroup
// each.
//
// Bound: no unit, but the chain scores -> P -> PV -> scores with its waits.  32 trees of 64 nodes
// over 2048 keys (70.9 GFLOP, 173 MB): 137 to 143 us by card, where the matrix products alone would
// take 42 and the bytes 27.  128 keys against 256 rows take a CTA about 5.5 thousand cycles, of
// which the tensor core works 2.1 and 16 softmax warps beside four converters 3.5 in a loop of
// their own.  That is not what such trees have to cost: the 16-bit cache's kernel takes 112 us on
// them (a serving mix: 326, here 473).  Work that it does not have: the key factors in both passes
// over the scores, the expansion of V by four warps, and with one query tile half a key tile and an
// O per stream.  So the 8-bit cache saves bytes here, and time where the bytes count (long decode).
//
//   warps 0, 2   MMA issuers, one per stream; TMEM (S0, S1, O0, O1: 128 columns each)
//   warp 1       work pieces; TMA loads of K, V and scale bytes for prefix tiles
//   warp 3       cp.async gathers of tiles that touch tree nodes or pages TMA cannot box
//   warps 4-7    scale bytes -> key factors; V codes -> bf16 tile
//   warps 8-23   softmax + epilogue: a warpgroup per score buffer, a thread per row
//
// Every mbarrier wait is bounded; one that runs out sets JT_DEVERR_TIMEOUT and the CTA's
// abort flag, all roles leave their loops, drain what they started and free the TMEM.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <climits>

#include "common.cuh"

namespace {

__device__ uint32_t g_attn_fp8_errors;

constexpr int kN = 128;               // keys per tile
constexpr int kHalf = 64;             // keys per score buffer (a granule)
constexpr int kM = 128;               // rows per query tile
constexpr int kD = 128;               // head dim in shared memory (shorter heads: zeros)
constexpr int kThreads = 768;
constexpr int kKRing = 3, kVRing = 2;
// The scale bytes' ring: a slot is refilled with tile g + 8 once QK g + 5 has been issued, hence
// after PV g + 3, hence after the converters read tile g's.
constexpr int kScaleRing = 8;
constexpr int kTile8 = kN * kD;       // bytes of a code tile
constexpr int kTile16 = 2 * kTile8;   // bytes of a bf16 tile: two 64-dim halves
constexpr int kHalf16 = kTile8;
constexpr int kMaxCtas = 160;         // workspace slots are sized for this many SMs
constexpr int kMaxNodes = 1024;
constexpr int kFewRows = 16;          // requests with up to this many rows: tree_attn_fp8_few.cuh
constexpr int kMaskWords = kMaxNodes / 32;
// Costs of the work line: a key tile against one and against two query tiles, an item's fixed
// cost (pipeline fill, first maxima, epilogue), and the least part worth a CTA of its own.  From
// the CTAs' cycles over a mix of items: 4.2 thousand, 6.0 thousand and 13 to 17 thousand.
constexpr int kTileCost = 2, kPairCost = 3;
constexpr int kItemCost = 8;
constexpr int kMinPart = 12;          // one request of 500 keys and 64 nodes: 42 us, 60 with 24
constexpr int kMinTiles = 2;          // cuts closer than this to an item's end move to it
constexpr long long kWaitLimit = 4000000000ll;  // cycles (~2 s) per wait

// ---- shared memory ------------------------------------------------------------------
template <bool kWide>
struct Smem {
  static constexpr int kTerms = kWide ? 3 : 2;   // e4m3 terms of a query element
  static constexpr int kTiles = kWide ? 1 : 2;   // query tiles per item
  static constexpr int kQ = 0;
  static constexpr int kK = kQ + kTiles * kTerms * kTile8;
  static constexpr int kV8 = kK + kKRing * kTile8;
  static constexpr int kV16 = kV8 + kVRing * kTile8;
  static constexpr int kScale = kV16 + 2 * kTile16;          // [kScaleRing][K, V][128] bytes
  static constexpr int kLost = kScale + kScaleRing * 256;     // [kScaleRing][4] words: keys without a place
  static constexpr int kKf = kLost + kScaleRing * 16;         // [2][128] float
  static constexpr int kX = kKf + 2 * kN * 4;                 // [stream][half][128] float2: max, sum
  static constexpr int kMx = kX + 4 * kM * 8;                 // [stream][128] float: maxima
  static constexpr int kItem = kMx + 2 * kM * 4;              // [2][16] int
  static constexpr int kFlag = kItem + 2 * 64;                // [2][4] int2: rare forms; keys without a place
  static constexpr int kMisc = kFlag + 64;                    // TMEM base, abort, free slots
  static constexpr int kBar = kMisc + 32;
  static constexpr int kBytes = kBar + 8 * 64 + 1024;         // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory per CTA");
};

// ---- barriers -------------------------------------------------------------------------
constexpr int kBarKFull = 0;     // [3] TMA (arrive_tx) or the gather warp
constexpr int kBarKEmpty = 3;    // [3] commit after each stream's last QK of the tile
constexpr int kBarVFull = 6;     // [2] TMA or the gather warp
constexpr int kBarVEmpty = 8;    // [2] 4 converter warps
constexpr int kBarFac = 10;      // [2] 4 converter warps: the tile's factors are written
constexpr int kBarBFull = 12;    // [2] 4 converter warps: the tile's bf16 V is written
constexpr int kBarBEmpty = 14;   // [2] commit after each stream's last PV of the tile
constexpr int kBarQEmpty = 16;   // commit after each stream's last QK of a piece
constexpr int kBarODone = 17;    // commit after each stream's last PV of a piece
constexpr int kBarQFull = 18;    // TMA
constexpr int kBarSFull = 19;    // [2 streams][2 buffers] commit per QK
constexpr int kBarPFull = 23;    // [2 streams][2 buffers] 4 softmax warps
constexpr int kBarPv = 27;       // [2] commit per PV, by stream
constexpr int kBarOFree = 29;    // 16 softmax warps: the epilogue has read O
constexpr int kBarX = 30;        // 16 softmax warps: (max, sum) exchanged
constexpr int kBarItemEmpty = 31;  // [2] every warp
constexpr int kBarItemFull = 33;   // [2] publisher
constexpr int kBarDrain = 35;      // [2] commit after a stream's last MMA
constexpr int kBarMx = 37;         // [stream][buffer][32 rows] the warp has set the rows' maxima
constexpr int kBarScale = 53;      // [8] as KFull, for the tile's scale bytes
constexpr int kNumBars = 61;
static_assert(kNumBars <= 64, "barrier area");

__device__ __forceinline__ uint32_t bar_count(int i) {
  if (i < kBarKEmpty) return 1;
  if (i < kBarVFull) return 2;   // KEmpty
  if (i < kBarVEmpty) return 1;
  if (i < kBarBEmpty) return 4;  // VEmpty, Fac, BFull
  if (i < kBarQFull) return 2;   // BEmpty, QEmpty, ODone
  if (i < kBarPFull) return 1;   // QFull, SFull
  if (i < kBarPv) return 4;
  if (i < kBarOFree) return 1;   // Pv
  if (i < kBarItemEmpty) return 16;
  return i < kBarItemFull ? kThreads / 32 : 1;
}

// TMEM columns.
__device__ __forceinline__ constexpr uint32_t col_s(int s, int b) { return 128u * s + 64u * b; }
__device__ __forceinline__ constexpr uint32_t col_o(int s) { return 256u + 128u * s; }

// ---- PTX ------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort,
                                            bool abortable) {
  const long long start = clock64();
  for (;;) {
    if (mbar_try(bar, parity)) return true;
    if (abortable && *abort) return false;
    if (clock64() - start > kWaitLimit) {
      *abort = 1;
      atomicOr(&g_attn_fp8_errors, JT_DEVERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, volatile int* abort,
                                          bool abortable = true) {
  if (mbar_try(bar, parity)) return true;
  return mbar_wait_slow(bar, parity, abort, abortable);
}
__device__ __forceinline__ void warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  mbar_wait(bar, parity, abort);
  __syncwarp();
}
__device__ __forceinline__ void warp_arrive(uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Release store / bounded acquire wait on a counter in shared memory that only grows (a
// difference below 2^31 counts as reached).
__device__ __forceinline__ void st_release_shared(uint32_t addr, uint32_t v) {
  asm volatile("st.release.cta.shared::cta.u32 [%0], %1;\n" ::"r"(addr), "r"(v) : "memory");
}
__device__ __noinline__ void wait_shared_at_least(uint32_t addr, uint32_t target,
                                                  volatile int* abort) {
  const long long start = clock64();
  for (;;) {
    uint32_t v;
    asm volatile("ld.acquire.cta.shared::cta.u32 %0, [%1];\n" : "=r"(v) : "r"(addr) : "memory");
    if (static_cast<int>(v - target) >= 0 || *abort) return;
    if (clock64() - start > kWaitLimit) {
      *abort = 1;
      atomicOr(&g_attn_fp8_errors, JT_DEVERR_TIMEOUT);
      return;
    }
  }
}
__device__ __forceinline__ void fence_proxy_async() {
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
}
// One lane of a full warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n selp.u32 %0, 1, 0, e;\n}\n" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                       uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
}
// Shared-memory matrix descriptor, 128-byte swizzle (sm_100 descriptor version 1).
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  uint64_t d = static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16;
  d |= static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}
// Instruction descriptors, fp32 accumulator: M128 N64, e4m3 x e4m3 (both K-major), and M128
// N128, bf16 x bf16 with an MN-major B.
constexpr uint32_t kIdescQK = (1u << 4) | (static_cast<uint32_t>(kHalf >> 3) << 17) |
                              (static_cast<uint32_t>(kM >> 4) << 24);
constexpr uint32_t kIdescPV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) |
                              (static_cast<uint32_t>(kD >> 3) << 17) |
                              (static_cast<uint32_t>(kM >> 4) << 24);

#define JT_LD32_REGS(v)                                                                      \
  "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),        \
      "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),             \
      "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),          \
      "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),          \
      "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]),          \
      "=r"(v[31])
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : JT_LD32_REGS(v)
      : "r"(taddr));
}
#undef JT_LD32_REGS
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15}, [%16];\n"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]),
        "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
        "=r"(v[14]), "=r"(v[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16};\n" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
      "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]),
                 "=r"(v[6]), "=r"(v[7])
               : "r"(taddr));
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t (&v)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::
          "r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// ---- numbers --------------------------------------------------------------------------
// 2^(byte - 127); byte 255 is NaN, byte 0 the subnormal 2^-127.
__device__ __forceinline__ float scale_value(uint32_t b) {
  if (b == 255u) return __uint_as_float(0x7fc00000u);
  return b == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(b << 23);
}
// Multipliers that take a code widened by widen() to its value in bf16: 2^(120 + byte - 127),
// as a product of two where that exceeds bf16's range.  A NaN scale gives zero: the V row is
// kept out of the product, and the key's score is NaN for the rows that see it.
__device__ __forceinline__ uint2 v_multipliers(uint32_t b) {
  if (b == 255u) return make_uint2(0u, 0x3f803f80u);
  const int k = static_cast<int>(b) - 7;  // 120 + b - 127
  const int e1 = min(k, 127), e2 = k - e1;
  const uint32_t m1 = static_cast<uint32_t>(e1 + 127) << 7, m2 = static_cast<uint32_t>(e2 + 127) << 7;
  return make_uint2(m1 | (m1 << 16), m2 | (m2 << 16));
}
// Four e4m3 codes as bf16 pairs of value * 2^-120: the code's exponent and mantissa fields
// dropped into bf16's (subnormal codes become bf16 subnormals of the same value).  The pairs
// are codes (0, 2) and (1, 3), which saves the byte permutes: the V tile's columns, and so O's,
// hold the head dims in the order 0, 2, 1, 3 of every four, undone where O is written out.  A NaN
// code (0x7f, 0xff), which this package's writer never makes, comes out as 480.  set_nan_codes puts
// the NaN where it belongs in tiles whose keys every row sees; in the others it would reach the
// rows that do not see the key as 0 x NaN: there the merge kernel gives it to the rows that do.
__device__ __forceinline__ void widen(uint32_t w, uint32_t& even, uint32_t& odd) {
  even = (w & 0x007f007fu) * 16u + (w & 0x00800080u) * 256u;
  odd = ((w >> 4) & 0x07f007f0u) | (w & 0x80008000u);
}
// The high bit of the bytes that hold a NaN code (other bits: noise).
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return (w & 0x7f7f7f7fu) + 0x01010101u; }
__device__ __forceinline__ uint32_t nan_codes(uint4 w) {
  return (nan_codes(w.x) | nan_codes(w.y) | nan_codes(w.z) | nan_codes(w.w)) & 0x80808080u;
}
// NaN where the codes of a converter warp's 32 V rows are NaN, in their bf16 rows: a row per lane.
__device__ __noinline__ void set_nan_codes(const unsigned char* src, unsigned char* dst) {
  const int row = threadIdx.x & 31;
#pragma unroll 1
  for (int c = 0; c < 16; ++c) {  // eight codes: two words
    const uint2 w = *reinterpret_cast<const uint2*>(src + row * 128 + (((c >> 1) ^ (row & 7)) << 4) + 8 * (c & 1));
    const uint32_t t[2] = {nan_codes(w.x), nan_codes(w.y)};
    uint4* o = reinterpret_cast<uint4*>(dst + (c >> 3) * kHalf16 + row * 128 + (((c & 7) ^ (row & 7)) << 4));
    if (((t[0] | t[1]) & 0x80808080u) == 0) continue;
    uint4 v = *o;
    v.x |= ((t[0] >> 7) & 0x00010001u) * 0x7fffu;
    v.y |= ((t[0] >> 15) & 0x00010001u) * 0x7fffu;
    v.z |= ((t[1] >> 7) & 0x00010001u) * 0x7fffu;
    v.w |= ((t[1] >> 15) & 0x00010001u) * 0x7fffu;
    *o = v;
  }
}
__device__ __forceinline__ constexpr int o_column(int d) {  // column of head dim d in O
  return (d & ~3) | ((d & 1) << 1) | ((d >> 1) & 1);
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t clamp_bf16x2(uint32_t a) {
  uint32_t r;
  asm("{\n .reg .b32 t;\n min.bf16x2 t, %1, %2;\n max.bf16x2 %0, t, %3;\n}\n"
      : "=r"(r)
      : "r"(a), "r"(0x7f7f7f7fu), "r"(0xff7fff7fu));
  return r;
}
__device__ __forceinline__ uint32_t pack_e4m3(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack_e4m3(uint32_t pair) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(h) : "h"(static_cast<uint16_t>(pair)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  return jt::MmaOp<__nv_bfloat16>::pack(lo, hi);
}

// ---- the work line ----------------------------------------------------------------------
struct Geometry {
  int groups, npt, npi;  // nodes per query tile, per item
};
struct ItemInfo {
  int key_end, n, two, weight, cost;
};
__device__ __forceinline__ ItemInfo item_info(const Geometry& ge, int P, int T, int mb) {
  const int first = mb * ge.npi, last = min(T, first + ge.npi);
  ItemInfo it;
  it.key_end = P + last;
  it.n = (it.key_end + kN - 1) >> 7;
  it.two = last - first > ge.npt;
  it.weight = it.two ? kPairCost : kTileCost;
  it.cost = it.n * it.weight + kItemCost;
  return it;
}
// Whether T nodes from packed row q0 on leave the call's rows, or their square the request's share
// of the bias.
__device__ __forceinline__ bool astray(const JtTreeAttnFp8Params& p, int T, int q0, int64_t biases) {
  return T > 0 && (q0 < 0 || T > p.total_queries - q0 || static_cast<int64_t>(T) * T > biases);
}
// A request as the kernels take it: no nodes when it has none or is refused.
__device__ __noinline__ int2 load_request(const JtTreeAttnFp8Params& p, int r, bool flag) {
  // Loaded together: calls of this are a chain that short launches wait for.
  int P = __ldg(p.prefix_lens + r), T = __ldg(p.node_counts + r);
  const int q0 = __ldg(p.cu_seqlens_q + r);
  const int64_t b0 = __ldg(p.qq_bias_offsets + r), b1 = __ldg(p.qq_bias_offsets + r + 1);
  const int64_t capacity = static_cast<int64_t>(p.table_width) * p.block_size;
  if (T > kMaxNodes || astray(p, T, q0, b1 - b0)) T = 0;  // refused: clear_refused
  if (P < 0 || P > capacity) {
    if (flag) atomicOr(&g_attn_fp8_errors, JT_DEVERR_OUT_OF_RANGE);
    P = P < 0 ? 0 : static_cast<int>(capacity);
  }
  return make_int2(P, max(T, 0));
}
__device__ __forceinline__ int2 tree_request(const JtTreeAttnFp8Params& p, int r, bool flag) {
  int2 q = load_request(p, r, flag);
  if (q.y * p.groups <= kFewRows) q.y = 0;  // the other kernel's
  return q;
}
__device__ __noinline__ int64_t head_cost(const Geometry ge, int P, int T) {
  int64_t c = 0;
#pragma unroll 1
  for (int mb = 0; mb * ge.npi < T; ++mb) c += item_info(ge, P, T, mb).cost;
  return c;
}
// Tile of an item at which a cut at line position x falls.
__device__ __forceinline__ int cut_tile(const ItemInfo& it, int64_t start, int64_t x) {
  if (x <= start) return 0;
  if (x >= start + it.cost) return it.n;
  const int t = static_cast<int>(x - start) / it.weight;
  if (t < kMinTiles) return 0;
  if (it.n - t < kMinTiles) return it.n;
  return t;
}

struct Piece {
  int r, h, mb, P, T, q_start, t0, n, key_end, two, slot;
};
// A piece's partial slot in the workspace, or -1 for a whole item.
struct PieceMeta {
  int valid, finishes, r, h, mb;
  int nan;  // the CTA has met NaN codes of V in tiles with masked keys
  int pad[2];
};
struct Workspace {
  PieceMeta* meta;   // [2 * kMaxCtas]
  float2* ml;        // [slot][tile][128] max (log2 units), sum
  float4* o;         // [slot][tile][32 groups of 4 columns][128]
  float* q_factor;   // [kv head][packed query row] scale * log2(e) * 2^e
  uint32_t* mask;    // [node][kMaskWords] bit n: the node sees tree node n
  uint8_t* q_terms;  // [kv head][term][packed query row][128] e4m3
};
constexpr int64_t kMetaBytes = 2 * kMaxCtas * sizeof(PieceMeta);
constexpr int64_t kMlBytes = 2ll * kMaxCtas * 2 * kM * sizeof(float2);
constexpr int64_t kPartBytes = 2ll * kMaxCtas * 2 * kM * kD * sizeof(float);
static_assert(kMetaBytes % 256 == 0 && kMlBytes % 256 == 0, "workspace alignment");
// A packed query row is (node, query head of the group).
__host__ __device__ __forceinline__ int64_t factor_bytes(int64_t rows, int heads) {
  return (rows * heads * 4 + 255) / 256 * 256;
}
__host__ __device__ __forceinline__ int64_t mask_bytes(int64_t nodes) {
  return (nodes * kMaskWords * 4 + 255) / 256 * 256;
}
__host__ __device__ __forceinline__ Workspace carve(void* base, int64_t nodes = 0, int groups = 0,
                                                    int heads = 0) {
  char* b = static_cast<char*>(base);
  char* q = b + kMetaBytes + kMlBytes + kPartBytes;
  return Workspace{reinterpret_cast<PieceMeta*>(b), reinterpret_cast<float2*>(b + kMetaBytes),
                   reinterpret_cast<float4*>(b + kMetaBytes + kMlBytes), reinterpret_cast<float*>(q),
                   reinterpret_cast<uint32_t*>(q + factor_bytes(nodes * groups, heads)),
                   reinterpret_cast<uint8_t*>(q + factor_bytes(nodes * groups, heads) + mask_bytes(nodes))};
}

// Zeros for the rows of requests that no kernel of the launch takes, and the error bit that says
// why: what else they would hold is whatever lay in the caller's memory.  `least` and `most`: the
// rows that the launched kernels take.  A warp per CTA of the launch's last merge kernel, ahead of
// its wait (nothing else writes these rows): beside the attention's own warps it cost 2 to 3 %.
__device__ __noinline__ void clear_refused(const JtTreeAttnFp8Params& p, int least, int most) {
  const int lane = threadIdx.x & 31;
  const int64_t stride = gridDim.x;
  for (int64_t first = blockIdx.x; first < p.num_requests; first += 32 * stride) {
    const int64_t r = first + lane * stride;
    int T = 0, q0 = 0;
    int64_t biases = 0;
    if (r < p.num_requests) {
      T = __ldg(p.node_counts + r);
      q0 = __ldg(p.cu_seqlens_q + r);
      biases = __ldg(p.qq_bias_offsets + r + 1) - __ldg(p.qq_bias_offsets + r);
    }
    const bool large = T > kMaxNodes;
    const bool out = astray(p, T, q0, biases) ||
                     (T > 0 && !large && (T * p.groups < least || T * p.groups > most));
    if (large) atomicOr(&g_attn_fp8_errors, JT_DEVERR_TREE_TOO_LARGE);
    if (out) atomicOr(&g_attn_fp8_errors, JT_DEVERR_OUT_OF_RANGE);
    uint32_t todo = __ballot_sync(0xffffffffu, large || out);
    for (; todo != 0; todo &= todo - 1) {
      const int src = __ffs(todo) - 1;
      const int64_t q = __shfl_sync(0xffffffffu, q0, src), n = __shfl_sync(0xffffffffu, T, src);
      const int64_t lo = max(q, static_cast<int64_t>(0));
      const int64_t hi = min(q + n, static_cast<int64_t>(p.total_queries));
      const int heads = p.num_kv_heads * p.groups, size = p.out_dtype == JT_F32 ? 4 : 2;
      const int words = p.head_dim * size / 16;  // per head, 16 bytes each
      for (int64_t i = lane; i < (hi - lo) * heads * words; i += 32) {
        const int64_t row = i / (heads * words);
        const int rest = static_cast<int>(i - row * (heads * words)), head = rest / words;
        char* dst = static_cast<char*>(p.out) + ((lo + row) * p.out_stride0 + head * p.out_stride1) * size;
        reinterpret_cast<uint4*>(dst)[rest - head * words] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }
}

// Page and offset of key position `pos` of a piece, page -1 past its keys or out of the pool.
struct KeyPlace {
  int64_t page;
  int off;
};
__device__ __noinline__ KeyPlace locate_key(const JtTreeAttnFp8Params& p, const int32_t* table,
                                            int pos, int P, int key_end, int q_start) {
  KeyPlace k{-1, 0};
  if (pos >= key_end) return k;
  int64_t slot;
  if (pos < P) {
    const int col = pos / p.block_size;
    slot = static_cast<int64_t>(__ldg(table + col)) * p.block_size + (pos - col * p.block_size);
  } else {
    slot = __ldg(p.tree_slots + q_start + (pos - P));
  }
  if (slot >= 0 && slot < p.num_blocks * static_cast<int64_t>(p.block_size)) {
    k.page = slot / p.block_size;
    k.off = static_cast<int>(slot - k.page * p.block_size);
  } else {
    atomicOr(&g_attn_fp8_errors, JT_DEVERR_OUT_OF_RANGE);
  }
  return k;
}
// One row's 16-byte chunks into a swizzled code tile (zeros past `chunks` or without a page).
__device__ __noinline__ void gather_row(uint32_t dst, int row, const char* src, int chunks) {
#pragma unroll 1
  for (int c = 0; c < 8; ++c)
    jt::cp_async_16(dst + row * 128 + ((c ^ (row & 7)) << 4), c < chunks ? src + 16 * c : src,
                    c < chunks ? 16 : 0);
}

// V codes that are NaN in tiles with masked keys: whoever meets one notes it for the CTA's pieces,
// and the merge kernel makes NaN of the rows that see its key, node by node.  Asked in the
// attention's own epilogue the question took 3 % of a serving mix, asked in the few-row kernel's
// loop 1.5 % of a long decode.
__device__ __noinline__ void note_nan_codes(const JtTreeAttnFp8Params& p) {
  PieceMeta* m = carve(p.workspace).meta + 2 * blockIdx.x;
  m[0].nan = m[1].nan = 1;
}
__device__ __noinline__ bool sees_nan_code(const JtTreeAttnFp8Params& p, int r, int2 request, int h, int j) {
  const int P = request.x, q_start = __ldg(p.cu_seqlens_q + r), key_end = P + j + 1;
  const int32_t* table = p.block_tables + static_cast<int64_t>(r) * p.table_stride0;
  const float* bias = p.qq_bias + __ldg(p.qq_bias_offsets + r) + static_cast<int64_t>(j) * request.y;
#pragma unroll 1
  for (int pos = P / kN * kN; pos < key_end; ++pos) {
    if (pos >= P && bias[pos - P] != 0.f) continue;
    const KeyPlace at = locate_key(p, table, pos, P, key_end, q_start);
    if (at.page < 0) continue;
    const uint4* row = reinterpret_cast<const uint4*>(static_cast<const char*>(p.v_pool) + at.page * p.v_stride0 +
                                                      at.off * p.v_stride1 + h * p.v_stride2);
#pragma unroll 1
    for (int c = 0; c < p.head_dim / 16; ++c)
      if (nan_codes(row[c]) != 0) return true;
  }
  return false;
}
// The same for every node and KV head of the requests of `least` to `most` rows, by one block.
// Rows of cut items are merged by other blocks, which make NaN of the same ones.
__device__ __noinline__ void spread_nan_codes(const JtTreeAttnFp8Params& p, int least, int most) {
  const int size = p.out_dtype == JT_F32 ? 4 : 2, words = p.head_dim * size / 16;
#pragma unroll 1
  for (int r = 0; r < p.num_requests; ++r) {
    const int2 q = load_request(p, r, false);
    if (q.y * p.groups < least || q.y * p.groups > most) continue;
    const int64_t q_start = __ldg(p.cu_seqlens_q + r);
#pragma unroll 1
    for (int i = threadIdx.x; i < q.y * p.num_kv_heads; i += blockDim.x) {
      const int j = i / p.num_kv_heads, h = i - j * p.num_kv_heads;
      if (!sees_nan_code(p, r, q, h, j)) continue;
#pragma unroll 1
      for (int k = 0; k < p.groups * words; ++k) {
        const int head = h * p.groups + k / words;
        char* dst = static_cast<char*>(p.out) + ((q_start + j) * p.out_stride0 + head * p.out_stride1) * size;
        // NaN as one 32-bit value and as two of either 16-bit type.
        reinterpret_cast<uint4*>(dst)[k % words] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      }
    }
  }
}

// Marks keys lo to hi - 1 of a tile, in sixteens, as without a place in the pool.  Out of line,
// and the words are cleared by their reader: what the loading lane runs for every tile counts
// (words that it writes for each: 2.5 % of a serving mix).
__device__ __noinline__ void lose_keys(uint32_t words, int lo, int hi) {
  atomicOr(&g_attn_fp8_errors, JT_DEVERR_OUT_OF_RANGE);
#pragma unroll 1
  for (int k = lo; k < hi; k += 16)
    asm volatile("{\n .reg .b32 w;\n ld.shared.u32 w, [%0];\n or.b32 w, w, %1;\n st.shared.u32 [%0], w;\n}\n" ::"r"(
                     words + 4 * (k >> 5)),
                 "r"(0xffffu << (k & 31))
                 : "memory");
}

// How tiles reach shared memory, decided on the host from the layout.
struct LoadPlan {
  int tma;   // prefix tiles by TMA boxes of `box` keys, their scale bytes by bulk copies
  int box;
};

// Visibility words of 64 keys for a row, from its node's bits: bit b of the first word is the key
// `off` + b past the prefix.  Prefix keys are visible.
__device__ __noinline__ uint2 mask_words(const uint32_t* bits, int off) {
  uint32_t w[3], out[2];
  const int first = off >> 5;  // -1 and below: prefix
#pragma unroll
  for (int i = 0; i < 3; ++i)
    w[i] = first + i < 0 ? ~0u : first + i < kMaskWords ? __ldg(bits + first + i) : 0u;
#pragma unroll
  for (int i = 0; i < 2; ++i) out[i] = __funnelshift_r(w[i], w[i + 1], off & 31);
  return make_uint2(out[0], out[1]);
}

// The largest of a row's 64 scores (times the keys' factors) of a granule, and then, with the
// row's running maximum known, their probabilities.  The scores are read from TMEM twice, 32 at
// a time, rather than held: with 24 warps a thread has 80 registers, and four softmax warps per
// scheduler hide each other's latencies, which two with the scores in registers do not (the
// mix above 750 us with two, 615 with four).
__device__ __forceinline__ void load_scores(uint32_t s_addr, const float* kf, uint32_t (&v)[32]) {
  tmem_ld32(s_addr, v);
  tmem_wait_ld();
  const float4* f4 = reinterpret_cast<const float4*>(kf);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float4 f = f4[k];
    const float2 a = __fmul2_rn(make_float2(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1])),
                                make_float2(f.x, f.y));
    const float2 b = __fmul2_rn(make_float2(__uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3])),
                                make_float2(f.z, f.w));
    v[4 * k] = __float_as_uint(a.x);
    v[4 * k + 1] = __float_as_uint(a.y);
    v[4 * k + 2] = __float_as_uint(b.x);
    v[4 * k + 3] = __float_as_uint(b.y);
  }
}
__device__ __forceinline__ float half_max(uint32_t s_addr, const float* kf) {
  float mx = -INFINITY;
#pragma unroll 1
  for (int q = 0; q < 2; ++q) {
    uint32_t v[32];
    load_scores(s_addr + 32 * q, kf + 32 * q, v);
    float m8[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) m8[k] = fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 8]));
#pragma unroll
    for (int k = 0; k < 8; ++k)
      m8[k] = max3f(m8[k], __uint_as_float(v[k + 16]), __uint_as_float(v[k + 24]));
    mx = max3f(mx, max3f(m8[0], m8[1], m8[2]), max3f(m8[3], m8[4], m8[5]));
    mx = max3f(mx, m8[6], m8[7]);
  }
  return mx;
}
// P = exp2(score * c_row - m) as high and low bf16 parts, to the S columns the scores came from
// (the low parts 32 columns on); returns the fp32 sum.
__device__ __forceinline__ float half_exp_wide(uint32_t s_addr, const float* kf, float c_row, float neg_m) {
  const float2 c2 = make_float2(c_row, c_row), n2 = make_float2(neg_m, neg_m);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t low[16];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    uint32_t v[32], ph[16];
    load_scores(s_addr + 32 * q, kf + 32 * q, v);
    // The first low parts go where the second scores were.
    if (q == 1) tmem_st16(s_addr + 32, low);
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const float2 x = __ffma2_rn(
          make_float2(__uint_as_float(v[2 * k]), __uint_as_float(v[2 * k + 1])), c2, n2);
      const float2 e = make_float2(jt::fast_exp2(x.x), jt::fast_exp2(x.y));
      sum[k & 1] = __fadd2_rn(sum[k & 1], e);
      ph[k] = pack_bf16(e.x, e.y);
      const float2 f = jt::MmaOp<__nv_bfloat16>::unpack(ph[k]);
      low[k] = pack_bf16(e.x - f.x, e.y - f.y);
    }
    tmem_st16(s_addr + 16 * q, ph);
  }
  tmem_st16(s_addr + 48, low);
  return (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
}
// The same rounded to bf16, 16 columns at a time with the next 16 on their way (against 32 at a
// time: 3 % of a mix).
__device__ __forceinline__ float half_exp_narrow(uint32_t s_addr, const float* kf, float c_row, float neg_m) {
  const float2 c2 = make_float2(c_row, c_row), n2 = make_float2(neg_m, neg_m);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  uint32_t v[2][16];
  tmem_ld16(s_addr, v[0]);
  const float4* f4 = reinterpret_cast<const float4*>(kf);
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    tmem_wait_ld();
    if (c < 3) tmem_ld16(s_addr + 16 * (c + 1), v[(c + 1) & 1]);
    uint32_t ph[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float4 f = f4[4 * c + k];
      const uint32_t* x = v[c & 1] + 4 * k;
      const float2 xa = make_float2(__uint_as_float(x[0]), __uint_as_float(x[1]));
      const float2 xb = make_float2(__uint_as_float(x[2]), __uint_as_float(x[3]));
      const float2 a = __ffma2_rn(__fmul2_rn(xa, make_float2(f.x, f.y)), c2, n2);
      const float2 b = __ffma2_rn(__fmul2_rn(xb, make_float2(f.z, f.w)), c2, n2);
      const float2 ea = make_float2(jt::fast_exp2(a.x), jt::fast_exp2(a.y));
      const float2 eb = make_float2(jt::fast_exp2(b.x), jt::fast_exp2(b.y));
      sum[0] = __fadd2_rn(sum[0], ea);
      sum[1] = __fadd2_rn(sum[1], eb);
      ph[2 * k] = pack_bf16(ea.x, ea.y);
      ph[2 * k + 1] = pack_bf16(eb.x, eb.y);
    }
    tmem_st8(s_addr + 8 * c, ph);
  }
  return (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
}

// The same for tiles with masked keys, a NaN row or a key without a place in the pool (the last
// one or two of an item, and few others): masked scores are -inf, every exponential is exp2,
// which keeps a NaN.  Rolled over 8 columns: a few hundred instructions that run seldom cost
// more to fetch than to execute.
__device__ __noinline__ float half_max_masked(uint32_t s_addr, const float* kf, uint32_t m0,
                                              uint32_t m1) {
  float mx = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < 8; ++c) {
    uint32_t v[8];
    tmem_ld8(s_addr + 8 * c, v);
    tmem_wait_ld();
    const uint32_t bits = (c < 4 ? m0 : m1) >> (8 * (c & 3));
#pragma unroll
    for (int k = 0; k < 8; ++k)
      mx = fmaxf(mx, (bits >> k) & 1u ? __uint_as_float(v[k]) * kf[8 * c + k] : -INFINITY);
  }
  return mx;
}
template <bool kWide>
__device__ __noinline__ float half_exp_masked(uint32_t s_addr, const float* kf, float c_row,
                                              float neg_m, uint32_t m0, uint32_t m1) {
  float sum = 0.f;
  if constexpr (kWide) {
    uint32_t low[16];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t v[32], ph[16];
      load_scores(s_addr + 32 * q, kf + 32 * q, v);
      if (q == 1) tmem_st16(s_addr + 32, low);
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float e[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int col = 2 * k + i;
          const float x = ((q ? m1 : m0) >> col) & 1u ? __uint_as_float(v[col]) : -INFINITY;
          e[i] = jt::fast_exp2(fmaf(x, c_row, neg_m));
          sum += e[i];
        }
        ph[k] = pack_bf16(e[0], e[1]);
        const float2 f = jt::MmaOp<__nv_bfloat16>::unpack(ph[k]);
        low[k] = pack_bf16(e[0] - f.x, e[1] - f.y);
      }
      tmem_st16(s_addr + 16 * q, ph);
    }
    tmem_st16(s_addr + 48, low);
  } else {
#pragma unroll 1
    for (int c = 0; c < 8; ++c) {
      uint32_t v[8], ph[4];
      tmem_ld8(s_addr + 8 * c, v);
      tmem_wait_ld();
      const uint32_t bits = (c < 4 ? m0 : m1) >> (8 * (c & 3));
      float e[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float x = (bits >> k) & 1u ? __uint_as_float(v[k]) * kf[8 * c + k] : -INFINITY;
        e[k] = jt::fast_exp2(fmaf(x, c_row, neg_m));
        sum += e[k];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) ph[k] = pack_bf16(e[2 * k], e[2 * k + 1]);
      tmem_st4(s_addr + 4 * c, ph);  // over scores already read
    }
  }
  return sum;
}

// 16 output columns of one row.  The narrow kernel's output is bf16.
template <bool kWide>
__device__ __forceinline__ void store_columns(const JtTreeAttnFp8Params& p, int64_t at,
                                              const float (&o)[16]) {
  if (kWide && p.out_dtype == JT_F32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      dst[k] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
    return;
  }
  uint32_t w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e)
    w[e] = !kWide || p.out_dtype == JT_BF16 ? pack_bf16(o[2 * e], o[2 * e + 1])
                                            : jt::MmaOp<__half>::pack(o[2 * e], o[2 * e + 1]);
  uint16_t* dst = static_cast<uint16_t*>(p.out) + at;
  if ((reinterpret_cast<uintptr_t>(dst) & 31u) == 0) {  // a whole sector per lane
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(dst), "r"(w[0]),
                 "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  } else {
    reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
    reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// Four output columns of one row from its unnormalised sums, O / l 2^shift.
template <bool kWide>
__device__ __forceinline__ void store_row4(const JtTreeAttnFp8Params& p, int q_start, int h, int row,
                                           int d, float4 o, float l, float shift) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (l == 0.f) {  // the row sees no key
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    shift = 0.f;
  }
  // In two steps: 2^shift alone may leave fp32's range.
  const float g = jt::fast_exp2(0.5f * shift);
  o = make_float4(o.x * inv * g * g, o.y * inv * g * g, o.z * inv * g * g, o.w * inv * g * g);
  const int node = row / p.groups;
  const int64_t at = (static_cast<int64_t>(q_start) + node) * p.out_stride0 +
                     (static_cast<int64_t>(h) * p.groups + row - node * p.groups) * p.out_stride1 + d;
  if (kWide && p.out_dtype == JT_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) = o;
  } else {
    const bool bf = !kWide || p.out_dtype == JT_BF16;
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) =
        bf ? make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w))
           : make_uint2(jt::MmaOp<__half>::pack(o.x, o.y), jt::MmaOp<__half>::pack(o.z, o.w));
  }
}

// Queries as e4m3 terms of row / 2^e and the rows' factors, for the attention kernel's TMA: half
// a warp per row (16 bytes per lane), its largest magnitude by shuffles.  A kernel of its own
// (the attention starts beside it as a programmatic dependent): inside, the split of a
// piece's 256 rows by one warpgroup took 25 thousand cycles, a third of a short piece.  The
// blocks from `first_mask` on turn the nodes' bias rows into visibility bits, a warp per node:
// built at the start of a piece by its softmax warps, from the fp32 biases, they held up its
// first tile by 7 thousand cycles.
template <bool kWide, typename QT>
__global__ void __launch_bounds__(256) tree_attn_fp8_split_kernel(
    const __grid_constant__ JtTreeAttnFp8Params p, const unsigned first_mask) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (blockIdx.x >= first_mask) {
    const int64_t q = static_cast<int64_t>(blockIdx.x - first_mask) * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (q >= p.total_queries) return;
    const int r = __ldg(p.query_to_request + q), j = __ldg(p.query_local_row + q);
    uint32_t mine = 0;  // word `lane`
    if (r >= 0 && r < p.num_requests && j >= 0) {
      const int T = __ldg(p.node_counts + r);
      const int q0 = __ldg(p.cu_seqlens_q + r);
      const int64_t b0 = __ldg(p.qq_bias_offsets + r), b1 = __ldg(p.qq_bias_offsets + r + 1);
      if (j < T && T <= kMaxNodes && !astray(p, T, q0, b1 - b0)) {
        const float* bias = p.qq_bias + b0 + static_cast<int64_t>(j) * T;
#pragma unroll 4
        for (int w = 0; 32 * w <= j; ++w) {
          const int n = 32 * w + lane;
          const uint32_t word = __ballot_sync(0xffffffffu, n <= j && __ldg(bias + min(n, j)) == 0.f);
          if (lane == w) mine = word;
        }
      }
    }
    carve(p.workspace, p.total_queries, p.groups, p.num_kv_heads).mask[q * kMaskWords + lane] = mine;
    return;
  }
  constexpr int kTerms = Smem<kWide>::kTerms;
  const int64_t rows = static_cast<int64_t>(p.total_queries) * p.groups;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 16 + (threadIdx.x >> 4);
  const int hl = threadIdx.x & 15;
  const bool ok = id < rows * p.num_kv_heads;
  const int64_t node = (ok ? id : 0) / (p.num_kv_heads * p.groups);
  const int hq = static_cast<int>((ok ? id : 0) - node * (p.num_kv_heads * p.groups));
  const int h = hq / p.groups;
  const int64_t row = node * p.groups + (hq - h * p.groups);
  uint4 w = make_uint4(0u, 0u, 0u, 0u);
  if (ok && 8 * hl < p.head_dim)
    w = __ldg(reinterpret_cast<const uint4*>(static_cast<const QT*>(p.q) + node * p.q_stride0 +
                                             hq * p.q_stride1 + 8 * hl));
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
  // The operands' own bits order like their magnitudes.
  uint32_t top = __vmaxu2(__vmaxu2(a[0] & 0x7fff7fffu, a[1] & 0x7fff7fffu),
                          __vmaxu2(a[2] & 0x7fff7fffu, a[3] & 0x7fff7fffu));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (!ok) return;
  top = __float_as_uint(jt::MmaOp<QT>::unpack(max(top & 0xffffu, top >> 16)).x);
  const bool finite = top < 0x7f800000u;
  int e = 0;
  if (top != 0 && finite)
    e = max(static_cast<int>(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u), -126);
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  float2 x[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[k] = jt::MmaOp<QT>::unpack(a[k]);
    x[k] = make_float2(x[k].x * inv, x[k].y * inv);
  }
  const Workspace ws = carve(p.workspace, p.total_queries, p.groups, p.num_kv_heads);
  uint8_t* dst = ws.q_terms + (static_cast<int64_t>(h) * kTerms * rows + row) * kD + 8 * hl;
#pragma unroll
  for (int m = 0; m < kTerms; ++m) {
    uint32_t t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      t[k] = pack_e4m3(x[k].x, x[k].y);
      const float2 y = unpack_e4m3(t[k]);
      x[k] = make_float2(x[k].x - y.x, x[k].y - y.y);
    }
    *reinterpret_cast<uint2*>(dst + m * rows * kD) = make_uint2(t[0] | (t[1] << 16), t[2] | (t[3] << 16));
  }
  // A row with a non-finite element: its factor makes its scores NaN.
  if (hl == 0)
    ws.q_factor[h * rows + row] =
        finite ? p.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 + e) << 23)
               : __uint_as_float(0x7fc00000u);
}

template <bool kWide>
__global__ void __launch_bounds__(kThreads, 1)
    tree_attn_fp8_kernel(const __grid_constant__ JtTreeAttnFp8Params p,
                         const __grid_constant__ CUtensorMap kmap,
                         const __grid_constant__ CUtensorMap vmap,
                         const __grid_constant__ CUtensorMap qmap, const LoadPlan plan) {
  using L = Smem<kWide>;
  constexpr int kTerms = L::kTerms;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = jt::smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* sbase = smem_raw + (base - raw);
  const uint32_t bar0 = base + L::kBar;
#define JT_BAR(i) (bar0 + 8u * static_cast<uint32_t>(i))
  volatile int* misc = reinterpret_cast<volatile int*>(sbase + L::kMisc);
  volatile int* abort = misc + 1;
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
  const Geometry ge{p.groups, kM / p.groups, (kM / p.groups) * L::kTiles};

  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  if (tid == 0) misc[1] = misc[2] = misc[3] = 0;
  if (tid < 4 * kScaleRing) reinterpret_cast<uint32_t*>(sbase + L::kLost)[tid] = 0;
  if (tid < kNumBars) {
    mbar_init(JT_BAR(tid), bar_count(tid));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    fence_proxy_async();
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(
                     base + L::kMisc)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }

  // This CTA's part of the work line: a block-wide scan of the requests' costs (a contiguous
  // run of requests per thread), then the request that holds the part's start.
  int64_t* scan = reinterpret_cast<int64_t*>(sbase + L::kV16);  // not in use yet
  const int R = p.num_requests, per = (R + kThreads - 1) / kThreads;
  const int r_lo = min(tid * per, R), r_hi = min(r_lo + per, R);
  int64_t mine = 0;
  for (int r = r_lo; r < r_hi; ++r) {
    const int2 q = tree_request(p, r, blockIdx.x == 0);
    mine += head_cost(ge, q.x, q.y) * p.num_kv_heads;
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
  for (int k = 0; k < kThreads / 32; ++k) {
    if (k < warp) before += scan[k];
    total += scan[k];
  }
  const int64_t my_start = before + incl - mine;
  const int parts = static_cast<int>(
      max(static_cast<int64_t>(1), min(static_cast<int64_t>(gridDim.x), total / kMinPart)));
  const bool has_part = static_cast<int>(blockIdx.x) < parts && total > 0;
  const int64_t x0 = has_part ? total * blockIdx.x / parts : 0;
  const int64_t x1 = has_part ? total * (blockIdx.x + 1) / parts : 0;
  if (has_part && mine > 0 && my_start <= x0 && x0 < my_start + mine) {
    int64_t s = my_start;
    for (int r = r_lo; r < r_hi; ++r) {
      const int2 q = tree_request(p, r, false);
      const int64_t c = head_cost(ge, q.x, q.y) * p.num_kv_heads;
      if (x0 < s + c) {
        scan[32] = r;
        scan[33] = s;
        break;
      }
      s += c;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, static_cast<uint32_t>(misc[0]), 0);
  const int r_start = has_part ? static_cast<int>(scan[32]) : R;
  const int64_t s_start = has_part ? scan[33] : 0;
  __syncthreads();  // the scan area is free
  // From here on the query terms are complete, and so is every earlier use of the workspace.
  asm volatile("griddepcontrol.wait;\n" ::: "memory");

  // Pieces: a two-entry ring in shared memory, filled one piece ahead by warp 1's first lane.
  volatile int* item_ring = reinterpret_cast<volatile int*>(sbase + L::kItem);
  auto next_piece = [&](uint32_t seq, Piece& it) -> bool {
    const int slot = seq & 1;
    int ok = 0;
    if (mbar_wait(JT_BAR(kBarItemFull + slot), (seq >> 1) & 1, abort) && !*abort) {
      volatile int* e = item_ring + 16 * slot;
      it.r = e[0]; it.h = e[1]; it.mb = e[2]; it.P = e[3]; it.T = e[4]; it.q_start = e[5];
      it.t0 = e[6]; it.n = e[7]; it.key_end = e[8]; it.two = e[9]; it.slot = e[10];
      ok = e[11];
    }
    ok = __all_sync(0xffffffffu, ok != 0);
    if (lane == 0) mbar_arrive(JT_BAR(kBarItemEmpty + slot));
    return ok != 0;
  };

  if (warp < 4) {
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------------------------- MMA issuers
      // One per stream: a step's waits, 12 MMAs and commits take a lone issuer, between warps
      // that keep every scheduler busy, longer than the softmax takes for the granule.
      const int s = warp >> 1;
      uint32_t g0 = 0, seq = 0;
      uint32_t p_phase = 0;  // bit b: score buffer b
      const uint64_t q_desc = smem_desc(base + L::kQ, 16, 1024);
      const uint64_t k_desc = smem_desc(base + L::kK, 16, 1024);
      const uint64_t v_desc = smem_desc(base + L::kV16, kHalf16, 1024);
      const uint32_t d_o = tmem + col_o(s);
      for (;; ++seq) {
        Piece it;
        if (!next_piece(seq, it)) break;
        const int n = __shfl_sync(0xffffffffu, it.n, 0), two = __shfl_sync(0xffffffffu, it.two, 0);
        mbar_wait(JT_BAR(kBarQFull), seq & 1, abort);
        tc_fence_after();
        // A stream takes its keys 64 at a time, in granules that alternate between its two
        // score buffers: with two query tiles granule k is half k & 1 of key tile k >> 1, with
        // one it is stream s's half of key tile k.  QK of granule k + 2 follows PV of granule
        // k, which read P out of the same buffer (MMAs of one thread execute in order);
        // granule k + 1 is in the softmax meanwhile.
        const int granules = two ? 2 * n : n;
        const uint64_t qd = q_desc + (two & s) * (kTerms * kTile8 / 16);
#pragma unroll 1
        for (int k = -2; k < granules; ++k) {
          const int b = k & 1, h = two ? b : s;
          const bool first = !two || b == 0, last = !two || b == 1;  // granule of its tile
          const uint32_t d_s = tmem + col_s(s, b);
          if (k >= 0) {
            const uint32_t g = g0 + (two ? k >> 1 : k);
            if (first) mbar_wait(JT_BAR(kBarBFull + (g & 1)), (g >> 1) & 1, abort);
            if (k == 0 && seq > 0) mbar_wait(JT_BAR(kBarOFree), (seq - 1) & 1, abort);
            mbar_wait(JT_BAR(kBarPFull + 2 * s + b), (p_phase >> b) & 1, abort);
            p_phase ^= 1u << b;
            tc_fence_after();
            const uint64_t vd = v_desc + ((g & 1) * kTile16 + h * (kHalf * 128)) / 16;
            if (elect_one()) {
#pragma unroll
              for (int kk = 0; kk < kHalf / 16; ++kk) {
                mma_ts(d_o, d_s + 8 * kk, vd + kk * (2048 / 16), kIdescPV, k > 0 || kk > 0 ? 1u : 0u);
                if constexpr (kWide)
                  mma_ts(d_o, d_s + 8 * kk + 32, vd + kk * (2048 / 16), kIdescPV, 1u);
              }
              commit(JT_BAR(kBarPv + s));
              if (last) commit(JT_BAR(kBarBEmpty + (g & 1)));
            }
            __syncwarp();
          }
          if (k + 2 < granules) {
            const int t = two ? (k + 2) >> 1 : k + 2;
            const uint32_t g = g0 + t;
            if (first) {
              mbar_wait(JT_BAR(kBarKFull + g % kKRing), (g / kKRing) & 1, abort);
              tc_fence_after();
            }
            const uint64_t kd = k_desc + ((g % kKRing) * kTile8 + h * (kHalf * 128)) / 16;
            if (elect_one()) {
#pragma unroll
              for (int m = 0; m < kTerms * 4; ++m)  // (term, 32 dims)
                mma_f8(d_s, qd + (m >> 2) * (kTile8 / 16) + (m & 3) * 2, kd + (m & 3) * 2, kIdescQK,
                       m != 0 ? 1u : 0u);
              commit(JT_BAR(kBarSFull + 2 * s + b));
              if (last) commit(JT_BAR(kBarKEmpty + g % kKRing));
              if (last && t == n - 1) commit(JT_BAR(kBarQEmpty));
            }
            __syncwarp();
          }
        }
        if (elect_one()) commit(JT_BAR(kBarODone));
        __syncwarp();
        g0 += n;
      }
      if (elect_one()) commit(JT_BAR(kBarDrain + s));
      __syncwarp();
      mbar_wait(JT_BAR(kBarDrain + s), 0, abort, false);
    } else if (warp == 1) {
      // ---------------------------------------------------------------- pieces and TMA
      // The whole warp follows the pieces; its first lane does the work.
      int r = r_start, h = 0, mb = 0, P = 0, T = 0;
      int64_t s_item = s_start;
      bool more = has_part;
      int meta_valid[2] = {0, 0};
      if (lane == 0 && more) {
        const int2 q = tree_request(p, r, false);
        P = q.x;
        T = q.y;
        const int64_t ch = head_cost(ge, P, T);
        h = static_cast<int>((x0 - s_item) / ch);
        s_item += ch * h;
        for (;;) {
          const ItemInfo it = item_info(ge, P, T, mb);
          if (x0 < s_item + it.cost) break;
          s_item += it.cost;
          ++mb;
        }
      }
      auto publish = [&](uint32_t seq) {
        const int slot = seq & 1;
        if (seq >= 2) mbar_wait(JT_BAR(kBarItemEmpty + slot), ((seq >> 1) - 1) & 1, abort);
        volatile int* e = item_ring + 16 * slot;
        e[11] = 0;
        while (more && !*abort) {
          const ItemInfo it = item_info(ge, P, T, mb);
          const int tb = cut_tile(it, s_item, x0), te = cut_tile(it, s_item, x1);
          const bool found = te > tb;
          if (found) {
            const bool whole = tb == 0 && te == it.n;
            const int which = tb == 0 ? 1 : 0;
            const int part = whole ? -1 : 2 * static_cast<int>(blockIdx.x) + which;
            e[0] = r; e[1] = h; e[2] = mb; e[3] = P; e[4] = T;
            e[5] = __ldg(p.cu_seqlens_q + r);
            e[6] = tb; e[7] = te - tb; e[8] = it.key_end; e[9] = it.two;
            e[10] = part; e[11] = 1;
            if (!whole) {
              PieceMeta* m = carve(p.workspace).meta + part;
              m->finishes = te == it.n;
              m->r = r;
              m->h = h;
              m->mb = mb;
              meta_valid[which] = 1;
            }
          }
          // On to the next item of the line.
          s_item += it.cost;
          if (s_item >= x1) {
            more = false;
          } else {
            ++mb;
            if (mb * ge.npi >= T) {
              mb = 0;
              if (++h == p.num_kv_heads) {
                h = 0;
                do {
                  ++r;
                  if (r < R) {
                    const int2 q = tree_request(p, r, false);
                    P = q.x;
                    T = q.y;
                  }
                } while (r < R && T == 0);
                if (r >= R) more = false;
              }
            }
          }
          if (found) break;
        }
        mbar_arrive(JT_BAR(kBarItemFull + slot));
      };
      uint32_t g0 = 0, q_fills = 0;
      // Full barriers whose last fill is TMA's, as bits (K 0.., V 4.., scales 8..), and the
      // phase parity of that fill: what the drain waits for.
      uint32_t mine = 0, parity = 0;
      auto note = [&](int bit, bool by_tma, uint32_t phase) {
        mine = (mine & ~(1u << bit)) | (by_tma ? 1u << bit : 0u);
        parity = (parity & ~(1u << bit)) | ((phase & 1u) << bit);
      };
      if (lane == 0) {
        PieceMeta* m = carve(p.workspace).meta + 2 * blockIdx.x;
        m[0].nan = m[1].nan = 0;
        publish(0);
      }
      const char* ksc = static_cast<const char*>(p.k_scale);
      const char* vsc = static_cast<const char*>(p.v_scale);
      for (uint32_t seq = 0;; ++seq) {
        Piece it;
        if (!next_piece(seq, it)) break;
        const int n = it.n;
        const int32_t* table = p.block_tables + static_cast<int64_t>(it.r) * p.table_stride0;
        auto load = [&](bool is_v, int t) {
          const int kb = (it.t0 + t) * kN;
          const uint32_t g = g0 + t;
          const int ring = is_v ? kVRing : kKRing;
          const int slot = g % ring;
          // This lane alone waits on the rings' empty barriers, for every tile in order: a
          // parity wait is right only for a waiter that is at most one phase behind.
          if (g >= static_cast<uint32_t>(ring))
            mbar_wait(JT_BAR((is_v ? kBarVEmpty : kBarKEmpty) + slot), ((g / ring) & 1) ^ 1, abort);
          if (*abort) return;
          if (!plan.tma || kb + kN > it.P) {  // gathered by warp 3, told that the slot is free
            note(is_v ? 4 + slot : slot, false, 0);
            if (!is_v) note(8 + g % kScaleRing, false, 0);
            st_release_shared(base + L::kMisc + (is_v ? 12 : 8), g + 1);
            return;
          }
          const uint32_t full = JT_BAR((is_v ? kBarVFull : kBarKFull) + slot);
          const uint32_t dst = base + (is_v ? L::kV8 : L::kK) + slot * kTile8;
          const uint32_t sc_slot = g % kScaleRing, sc_full = JT_BAR(kBarScale + sc_slot);
          mbar_arrive_tx(full, kTile8);
          if (!is_v) mbar_expect_tx(sc_full, 2 * kN);
#pragma unroll 1
          for (int i = 0; i < kN; i += plan.box) {
            const int pos = kb + i, off = pos % p.block_size;
            int page = __ldg(table + pos / p.block_size);
            if (page < 0 || page >= p.num_blocks) {
              // The box's keys are left out.  Page -1 lies outside the map: zeros.
              lose_keys(base + L::kLost + 16 * sc_slot, i, is_v ? i : i + plan.box);
              page = -1;
            }
            tma_load_4d(dst + i * kD, is_v ? &vmap : &kmap, 0, it.h, off, page, full);
            if (!is_v) {
              const int64_t pg = max(page, 0);
              const uint32_t sdst = base + L::kScale + sc_slot * 256 + i;
              bulk_load(sdst, ksc + pg * p.ks_stride0 + it.h * p.ks_stride1 + off, plan.box, sc_full);
              bulk_load(sdst + kN, vsc + pg * p.vs_stride0 + it.h * p.vs_stride1 + off, plan.box, sc_full);
            }
          }
          note(is_v ? 4 + slot : slot, true, g / ring);
          if (!is_v) {
            mbar_arrive(sc_full);  // with the missing keys written
            note(8 + sc_slot, true, g / kScaleRing);
          }
        };
        if (lane == 0) {
          // K 0, K 1, then V t and K t + 2: the order in which they are used.
#pragma unroll 1
          for (int i = 0; i <= 2 * n; ++i) {
            if (i == max(0, 2 * n - 6)) publish(seq + 1);
            if (i == 2) {
              // The query tiles, once the previous piece's last QK has read them.  Rows past
              // the item's are other nodes' (or zeros): their scores are never used.
              if (seq > 0) mbar_wait(JT_BAR(kBarQEmpty), (seq - 1) & 1, abort);
              const int tiles = 1 + it.two;
              mbar_arrive_tx(JT_BAR(kBarQFull), tiles * kTerms * kTile8);
              const int row = (it.q_start + it.mb * ge.npi) * ge.groups;
#pragma unroll 1
              for (int k = 0; k < tiles * kTerms; ++k)
                tma_load_3d(base + L::kQ + k * kTile8, &qmap, 0,
                            row + (k >= kTerms ? ge.npt * ge.groups : 0),
                            it.h * kTerms + (k >= kTerms ? k - kTerms : k), JT_BAR(kBarQFull));
              q_fills = seq + 1;
            }
            const bool is_v = i >= 2 && !(i & 1);
            const int t = i < 2 ? i : is_v ? (i >> 1) - 1 : (i >> 1) + 1;
            if (t < n) load(is_v, t);
          }
        }
        __syncwarp();
        g0 += n;
      }
      if (lane == 0) {
        // The copies this lane started have landed before the CTA exits.
#pragma unroll 1
        for (int i = 0; i < 16; ++i)
          if (mine & (1u << i)) {
            const int bar = i < 4 ? kBarKFull + i : i < 8 ? kBarVFull + i - 4 : kBarScale + i - 8;
            mbar_wait(JT_BAR(bar), (parity >> i) & 1u, abort, false);
          }
        if (q_fills > 0) mbar_wait(JT_BAR(kBarQFull), (q_fills - 1) & 1, abort, false);
        PieceMeta* m = carve(p.workspace).meta + 2 * blockIdx.x;
        m[0].valid = meta_valid[0];
        m[1].valid = meta_valid[1];
      }
    } else {
      // ---------------------------------------------------------------- gathers
      // Tiles that TMA does not take: rows by cp.async, scale bytes by plain loads into the
      // same staging.
      const int chunks = p.head_dim / 16;
      uint32_t g0 = 0;
#pragma unroll 1
      for (uint32_t seq = 0;; ++seq) {
        Piece it;
        if (!next_piece(seq, it)) break;
        const int32_t* table = p.block_tables + static_cast<int64_t>(it.r) * p.table_stride0;
#pragma unroll 1
        for (int t = plan.tma ? max(0, it.P / kN - it.t0) : 0; t < it.n; ++t) {
          const uint32_t g = g0 + t;
          const uint32_t ks = g % kKRing, vs = g % kVRing;
          // Four keys per lane; their slots and scales are loaded together, before the slot is
          // free.
          const char* k_src[4];
          const char* v_src[4];
          uint32_t kb[4], vb[4];
          bool ok[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const KeyPlace at = locate_key(p, table, (it.t0 + t) * kN + 32 * i + lane, it.P, it.key_end, it.q_start);
            ok[i] = at.page >= 0;
            const int64_t page = ok[i] ? at.page : 0;
            k_src[i] = static_cast<const char*>(p.k_pool) + page * p.k_stride0 + at.off * p.k_stride1 + it.h * p.k_stride2;
            v_src[i] = static_cast<const char*>(p.v_pool) + page * p.v_stride0 + at.off * p.v_stride1 + it.h * p.v_stride2;
            kb[i] = vb[i] = 127;
            if (ok[i]) {
              kb[i] = __ldg(static_cast<const uint8_t*>(p.k_scale) + page * p.ks_stride0 +
                            it.h * p.ks_stride1 + at.off);
              vb[i] = __ldg(static_cast<const uint8_t*>(p.v_scale) + page * p.vs_stride0 +
                            it.h * p.vs_stride1 + at.off);
            }
          }
          wait_shared_at_least(base + L::kMisc + 8, g + 1, abort);
          wait_shared_at_least(base + L::kMisc + 12, g + 1, abort);
          __syncwarp();
          unsigned char* sc = sbase + L::kScale + (g % kScaleRing) * 256 + lane;
          uint32_t* lost = reinterpret_cast<uint32_t*>(sbase + L::kLost) + 4 * (g % kScaleRing);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            gather_row(base + L::kK + ks * kTile8, 32 * i + lane, k_src[i], ok[i] ? chunks : 0);
            gather_row(base + L::kV8 + vs * kTile8, 32 * i + lane, v_src[i], ok[i] ? chunks : 0);
            sc[32 * i] = static_cast<unsigned char>(kb[i]);
            sc[kN + 32 * i] = static_cast<unsigned char>(vb[i]);
            const uint32_t none = __ballot_sync(0xffffffffu, !ok[i]);
            if (none != 0 && lane == 0) lost[i] = none;
          }
          asm volatile("cp.async.wait_all;\n" ::: "memory");
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(JT_BAR(kBarKFull + ks));
            mbar_arrive(JT_BAR(kBarVFull + vs));
            mbar_arrive(JT_BAR(kBarScale + g % kScaleRing));
          }
        }
        g0 += it.n;
      }
    }
  } else if (warp < 8) {
    // ------------------------------------------------------------------ converters
    const int ct = tid - 128, cw = warp - 4;  // this thread's key; this warp's 32 rows
    uint32_t g0 = 0;
    float* kf = reinterpret_cast<float*>(sbase + L::kKf);
    int2* flag = reinterpret_cast<int2*>(sbase + L::kFlag);
    // V: eight lanes of a warp take four 16-byte chunks of rows r and r ^ 5, so that both the
    // swizzled loads and the swizzled stores of the eight touch different banks.
    const int quad = lane >> 3, sub = lane & 7;
    const int v_half = quad & 1, v_chunk = v_half * 4 + (sub & 3);
#pragma unroll 1
    for (uint32_t seq = 0;; ++seq) {
      Piece it;
      if (!next_piece(seq, it)) break;
#pragma unroll 1
      for (int t = 0; t < it.n; ++t) {
        const uint32_t g = g0 + t, buf = g & 1;
        // Factors of this thread's key, once the tile's scale bytes are here and the buffers
        // of tile g - 2 are free (its last PV has completed).
        warp_wait(JT_BAR(kBarScale + g % kScaleRing), (g / kScaleRing) & 1, abort);
        const unsigned char* sc = sbase + L::kScale + (g % kScaleRing) * 256 + ct;
        const uint32_t kb = sc[0], vb = sc[kN];
        uint32_t* lost_word = reinterpret_cast<uint32_t*>(sbase + L::kLost) + 4 * (g % kScaleRing) + cw;
        const uint32_t lost = *lost_word;
        if (g >= 2) warp_wait(JT_BAR(kBarBEmpty + buf), ((g >> 1) & 1) ^ 1, abort);
        kf[buf * kN + ct] = vb == 255u ? scale_value(255u) : scale_value(kb);
        const uint2 mine = v_multipliers(vb);
        const bool rare = lost != 0 || __any_sync(0xffffffffu, kb == 255u || vb == 255u);
        const bool big = __any_sync(0xffffffffu, vb > 134u);  // needs the second multiplier
        __syncwarp();
        if (lane == 0) {
          flag[buf * 4 + cw] = make_int2(rare, static_cast<int>(lost));
          if (lost != 0) *lost_word = 0;
        }
        warp_arrive(JT_BAR(kBarFac + buf));
        warp_wait(JT_BAR(kBarVFull + g % kVRing), (g / kVRing) & 1, abort);
        // This warp's 32 rows x 8 chunks in 8 rounds, four rounds' loads in flight at a time.
        const unsigned char* src = sbase + L::kV8 + (g % kVRing) * kTile8 + cw * (32 * 128);
        unsigned char* dst = sbase + L::kV16 + buf * kTile16 + v_half * kHalf16 + cw * (32 * 128);
        uint32_t nan = 0;
#pragma unroll 1
        for (int i0 = 0; i0 < 8; i0 += 4) {
          uint4 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pr = (quad >> 1) + 2 * (i & 1);
            const int row = ((i0 + i) >> 1) * 8 + ((sub & 4) ? (pr ^ 5) : pr);
            w[i] = *reinterpret_cast<const uint4*>(src + row * 128 + ((v_chunk ^ (row & 7)) << 4));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pr = (quad >> 1) + 2 * (i & 1);
            const int row = ((i0 + i) >> 1) * 8 + ((sub & 4) ? (pr ^ 5) : pr);
            const uint32_t m = __shfl_sync(0xffffffffu, mine.x, row);
            uint32_t o[8];
            nan |= nan_codes(w[i]);
            widen(w[i].x, o[0], o[1]);
            widen(w[i].y, o[2], o[3]);
            widen(w[i].z, o[4], o[5]);
            widen(w[i].w, o[6], o[7]);
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] = mul_bf16x2(o[k], m);
            if (big) {
              // Saturating: an infinity would reach rows that do not see this key.
              const uint32_t m2 = __shfl_sync(0xffffffffu, mine.y, row);
#pragma unroll
              for (int k = 0; k < 8; ++k) o[k] = clamp_bf16x2(mul_bf16x2(o[k], m2));
            }
            unsigned char* row_dst = dst + row * 128;
            const int c0 = 2 * (sub & 3);
            *reinterpret_cast<uint4*>(row_dst + ((c0 ^ (row & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
            *reinterpret_cast<uint4*>(row_dst + (((c0 + 1) ^ (row & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
          }
        }
        if (__any_sync(0xffffffffu, nan != 0)) {
          __syncwarp();  // the rows are other lanes' too
          if ((it.t0 + t + 1) * kN <= it.P)
            set_nan_codes(src, sbase + L::kV16 + buf * kTile16 + cw * (32 * 128));
          else
            note_nan_codes(p);
        }
        fence_proxy_async();
        warp_arrive(JT_BAR(kBarBFull + buf));
        if (lane == 0) mbar_arrive(JT_BAR(kBarVEmpty + g % kVRing));
      }
      g0 += it.n;
    }
  } else {
    // ------------------------------------------------------------------ softmax + epilogue
    const int wg = (warp - 8) >> 2, s = wg >> 1, buf = wg & 1;  // stream, score buffer
    const int row = (tid - 256) & 127;                          // query-tile row, TMEM lane
    const uint32_t lanes = static_cast<uint32_t>((row >> 5) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + col_s(s, buf);
    const uint32_t my_bar = JT_BAR(kBarMx + (2 * s + buf) * 4 + (warp & 3));
    const uint32_t other_bar = JT_BAR(kBarMx + (2 * s + (buf ^ 1)) * 4 + (warp & 3));
    const float* kf = reinterpret_cast<const float*>(sbase + L::kKf);
    const Workspace ws = carve(p.workspace, p.total_queries, ge.groups, p.num_kv_heads);
    float2* xch = reinterpret_cast<float2*>(sbase + L::kX);
    float* m_row = reinterpret_cast<float*>(sbase + L::kMx) + s * kM + row;
    const int local = row / ge.groups, head_in = row - local * ge.groups;
    uint32_t g0 = 0, own = 0, other = 0;  // tiles; granules of this buffer, of the other one
#pragma unroll 1
    for (uint32_t seq = 0;; ++seq) {
      Piece it;
      if (!next_piece(seq, it)) break;
      const int n = it.n;
      const int j = it.mb * ge.npi + (it.two ? s * ge.npt : 0) + local;
      const bool ok = local < ge.npt && j < it.T;
      const bool live = __any_sync(0xffffffffu, ok);
      const int granules = it.two ? 2 * n : n, half = it.two ? buf : s;
      // Tiles below floor(P / 128) need no mask.
      const int t_mask = max(0, it.P / kN - it.t0);
      float m_run = -INFINITY, l_run = 0.f;
      const float c_row =
          ok ? __ldg(ws.q_factor + (static_cast<int64_t>(it.h) * p.total_queries + it.q_start + j) * ge.groups + head_in)
             : 0.f;
#pragma unroll 1
      for (int k = buf; k < granules; k += 2) {
        const int t = it.two ? k >> 1 : k;
        const uint32_t g = g0 + t, step = own + (k >> 1);
        bool careful = t >= t_mask;
        uint2 w = make_uint2(~0u, ~0u);
        if (careful && live) {
          w = mask_words(ws.mask + (static_cast<int64_t>(it.q_start) + (ok ? j : 0)) * kMaskWords,
                         (it.t0 + t) * kN + kHalf * half - it.P);
          if (!ok) w = make_uint2(0u, 0u);
        }
        warp_wait(JT_BAR(kBarFac + (g & 1)), (g >> 1) & 1, abort);
        warp_wait(JT_BAR(kBarSFull + 2 * s + buf), step & 1, abort);
        tc_fence_after();
        if (live) {
          const float* f = kf + (g & 1) * kN + kHalf * half;
          const int4* rare = reinterpret_cast<const int4*>(sbase + L::kFlag + 32 * (g & 1));
          const int4 r0 = rare[half];
          w.x &= ~static_cast<uint32_t>(r0.y);
          w.y &= ~static_cast<uint32_t>(r0.w);
          careful |= (r0.x | r0.z) != 0;
          const float mx = c_row * (careful ? half_max_masked(s_addr, f, w.x, w.y) : half_max(s_addr, f));
          // The rows' running maximum goes from granule to granule, between the two warps that
          // share the rows.  It is lazy: it moves only when a granule exceeds it by 2^8, so P
          // stays below 2^8 and O is rarely rescaled.
          float m_old = -INFINITY;
          if (k > 0) {
            warp_wait(other_bar, (other + ((k - 1) >> 1)) & 1, abort);
            m_old = *m_row;
          }
          const bool moved = mx > m_old + 8.f;
          const float m_new = moved ? mx : m_old;
          *m_row = m_new;
          warp_arrive(my_bar);
          // This warp's sum is relative to the maximum at its previous granule.
          if (m_run != m_new && m_run != -INFINITY) l_run *= jt::fast_exp2(m_run - m_new);
          m_run = m_new;
          const float neg_m = m_new == -INFINITY ? 0.f : -m_new;
          l_run += careful ? half_exp_masked<kWide>(s_addr, f, c_row, neg_m, w.x, w.y)
                           : kWide ? half_exp_wide(s_addr, f, c_row, neg_m)
                           : half_exp_narrow(s_addr, f, c_row, neg_m);
          if (__any_sync(0xffffffffu, moved && m_old != -INFINITY)) {
            // Rescale O once PV of the stream's previous granule has completed.  The wait is for
            // exactly the latest phase: the PV before it completed ahead of this granule's
            // scores, which were issued behind it, and the next PV needs this granule's P.
            const float alpha = moved && m_old != -INFINITY ? jt::fast_exp2(m_old - m_new) : 1.f;
            warp_wait(JT_BAR(kBarPv + s), (own + other + k - 1) & 1, abort);
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
              uint32_t o[16];
              tmem_ld16(tmem + lanes + col_o(s) + 16 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st16(tmem + lanes + col_o(s) + 16 * c, o);
            }
          }
          tmem_wait_st();
        } else {
          warp_arrive(my_bar);
        }
        // A warp without a live row arrives too; its rows of P are never read out.
        tc_fence_before();
        warp_arrive(JT_BAR(kBarPFull + 2 * s + buf));
      }
      // Epilogue, once the piece's last PV has completed: the halves' sums meet, with one query
      // tile also the streams' (max, sum).  With one tile each warpgroup merges and writes 32
      // of the columns, with two 64 of its stream's.
      warp_wait(JT_BAR(kBarODone), seq & 1, abort);
      tc_fence_after();
      xch[wg * kM + row] = make_float2(m_run, l_run);
      warp_arrive(JT_BAR(kBarX));
      warp_wait(JT_BAR(kBarX), seq & 1, abort);
      if (live) {
        const bool pair = !it.two;
        // A sum without a maximum is zero, or a NaN that has to stay.
        auto joined = [&](float2 a, float2 b) {
          const float m = fmaxf(a.x, b.x);
          return make_float2(m, a.y * (a.x == -INFINITY ? 1.f : jt::fast_exp2(a.x - m)) +
                                    b.y * (b.x == -INFINITY ? 1.f : jt::fast_exp2(b.x - m)));
        };
        const int s0 = pair ? 0 : 2 * s;
        const float2 a = joined(xch[s0 * kM + row], xch[(s0 + 1) * kM + row]);
        float fa = 1.f, fb = 0.f, m = a.x, l = a.y;
        if (pair) {
          const float2 b = joined(xch[2 * kM + row], xch[3 * kM + row]);
          const float2 both = joined(a, b);
          m = both.x;
          l = both.y;
          fa = a.x == -INFINITY ? 0.f : jt::fast_exp2(a.x - m);
          fb = b.x == -INFINITY ? 0.f : jt::fast_exp2(b.x - m);
        }
        const int tile = pair ? 0 : s;
        if (it.slot >= 0) {
          if (ok && (pair ? wg == 0 : buf == 0))
            ws.ml[(it.slot * 2ll + tile) * kM + row] = make_float2(m, l);
        } else {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          fa *= inv;
          fb *= inv;
        }
        const int64_t out_row = (static_cast<int64_t>(it.q_start) + j) * p.out_stride0 +
                                (static_cast<int64_t>(it.h) * ge.groups + head_in) * p.out_stride1;
        const int c0 = pair ? 2 * wg : 4 * buf, c1 = c0 + (pair ? 2 : 4);
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {  // 16 columns
          uint32_t o0[16], o1[16];
          __syncwarp();
          tmem_ld16(tmem + lanes + col_o(tile) + 16 * c, o0);
#pragma unroll
          for (int k = 0; k < 16; ++k) o1[k] = 0u;
          if (pair) tmem_ld16(tmem + lanes + col_o(1) + 16 * c, o1);
          tmem_wait_ld();
          float f[16];
#pragma unroll
          for (int k = 0; k < 16; ++k)
            f[k] = __uint_as_float(o0[o_column(k)]) * fa + __uint_as_float(o1[o_column(k)]) * fb;
          if (ok && it.slot >= 0) {
            float4* dst = ws.o + ((it.slot * 2ll + tile) * 32 + 4 * c) * kM + row;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              dst[k * kM] = make_float4(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3]);
          } else if (ok && 16 * c < p.head_dim) {
            if (l == 0.f) {  // the row sees no key
#pragma unroll
              for (int k = 0; k < 16; ++k) f[k] = 0.f;
            }
            store_columns<kWide>(p, out_row + 16 * c, f);
          }
        }
      }
      __syncwarp();
      tc_fence_before();
      warp_arrive(JT_BAR(kBarOFree));
      g0 += n;
      own += (granules + 1 - buf) >> 1;
      other += (granules + buf) >> 1;
    }
  }
#undef JT_BAR
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 0)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
}

// Merge of items cut between CTAs: block (c, q) takes 16 columns of the item that begins in
// CTA c's part and ends in a later one, a row per thread.  Its pieces are slot 2c + 1, then
// slots 2(c + 1), 2(c + 2), ... up to the one that finishes it.
template <bool kWide>
__global__ void __launch_bounds__(kM) tree_attn_fp8_merge_kernel(
    const __grid_constant__ JtTreeAttnFp8Params p, const int parts, const int least) {
  if (blockIdx.y == 0 && threadIdx.x < 32) clear_refused(p, least, INT_MAX);
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  const Workspace w = carve(p.workspace);
  const int c = blockIdx.x, tile = blockIdx.y >> 3, cg0 = (blockIdx.y & 7) * 4, row = threadIdx.x;
  const PieceMeta first = w.meta[2 * c + 1];
  if (first.nan != 0 && blockIdx.y == 0) spread_nan_codes(p, kFewRows + 1, INT_MAX);
  if (!first.valid || first.finishes || 4 * cg0 >= p.head_dim) return;
  const int npt = kM / p.groups, npi = npt * Smem<kWide>::kTiles;
  const int T = p.node_counts[first.r];
  const int local = row / p.groups;
  const int j = first.mb * npi + tile * npt + local;
  if (local >= npt || j >= T) return;
  float acc[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) acc[k] = 0.f;
  float m = -INFINITY, l = 0.f;
  int nan = 0;
  for (int i = c; i < parts; ++i) {
    const int slot = i == c ? 2 * c + 1 : 2 * i;
    if (i != c && !w.meta[slot].valid) continue;  // a part shorter than the least cut
    nan |= w.meta[slot].nan;
    const float2 ml = w.ml[(slot * 2ll + tile) * kM + row];
    float4 o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = w.o[((slot * 2ll + tile) * 32 + cg0 + k) * kM + row];
    const float top = fmaxf(m, ml.x), ref = top == -INFINITY ? 0.f : top;
    const float fa = m == -INFINITY ? 0.f : jt::fast_exp2(m - ref);
    const float fb = ml.x == -INFINITY ? 0.f : jt::fast_exp2(ml.x - ref);
    // A row whose keys were all NaN has no maximum but a NaN sum, which has to stay.
    l = l * (m == -INFINITY ? 1.f : fa) + ml.y * (ml.x == -INFINITY ? 1.f : fb);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      acc[4 * k] = acc[4 * k] * fa + o[k].x * fb;
      acc[4 * k + 1] = acc[4 * k + 1] * fa + o[k].y * fb;
      acc[4 * k + 2] = acc[4 * k + 2] * fa + o[k].z * fb;
      acc[4 * k + 3] = acc[4 * k + 3] * fa + o[k].w * fb;
    }
    m = top;
    if (i != c && w.meta[slot].finishes) break;
  }
  if (nan != 0 && sees_nan_code(p, first.r, load_request(p, first.r, false), first.h, j))
    l = __uint_as_float(0x7fc00000u);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int h = first.h * p.groups + (row - local * p.groups);
  const int64_t at = (static_cast<int64_t>(p.cu_seqlens_q[first.r]) + j) * p.out_stride0 +
                     h * p.out_stride1 + 4 * cg0;
  float f[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) f[k] = l != 0.f ? acc[k] * inv : 0.f;
  store_columns<kWide>(p, at, f);
}

int64_t workspace_bytes(int64_t nodes, int groups, int heads) {  // for either kernel's terms
  return kMetaBytes + kMlBytes + kPartBytes + factor_bytes(nodes * groups, heads) +
         mask_bytes(nodes) + nodes * groups * heads * 3 * kD;
}

bool al16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult query{};
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &query) ==
            cudaSuccess &&
        query == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    return static_cast<PFN_cuTensorMapEncodeTiled_v12000>(nullptr);
  }();
  return fn;
}

// [blocks, block_size, heads, head_dim] bytes; a box is `box` keys of one head, 128 bytes wide
// (zeros past head_dim), in the MMA operands' 128-byte swizzle.
bool encode_pool(CUtensorMap* map, const JtTreeAttnFp8Params& p, const void* pool, int64_t s0,
                 int64_t s1, int64_t s2, int box) {
  auto encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.head_dim),
                              static_cast<cuuint64_t>(p.num_kv_heads),
                              static_cast<cuuint64_t>(p.block_size),
                              static_cast<cuuint64_t>(p.num_blocks)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(s2), static_cast<cuuint64_t>(s1),
                                 static_cast<cuuint64_t>(s0)};
  const cuuint32_t boxes[4] = {kD, 1, static_cast<cuuint32_t>(box), 1};
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(pool), dims, strides,
                boxes, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [kv heads x terms][packed query rows][128] e4m3, a box of 128 rows.
bool encode_queries(CUtensorMap* map, const void* terms, int64_t rows, int planes) {
  auto encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const cuuint64_t dims[3] = {kD, static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {kD, static_cast<cuuint64_t>(rows) * kD};
  const cuuint32_t box[3] = {kD, kM, 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(terms), dims, strides, box,
                elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Programmatic dependent launch: the grid may start beside its predecessor and waits for it
// (griddepcontrol.wait) before it touches what that one writes.
template <typename... Params, typename... Args>
int launch_dependent(void (*kernel)(Params...), dim3 grid, int threads, size_t smem,
                     cudaStream_t stream, const char* what, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return jt_cuda_check(cudaLaunchKernelEx(&cfg, kernel, args...), what);
}

#include "tree_attn_fp8_few.cuh"

template <bool kWide, typename QT>
int launch(const JtTreeAttnFp8Params& p, int sms, cudaStream_t stream) {
  // A captured launch is replayed with other node counts than today's: it covers all sizes.
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  int rc = jt_cuda_check(cudaStreamIsCapturing(stream, &capture), "cudaStreamIsCapturing");
  if (rc != JT_OK) return rc;
  const bool known = p.max_nodes > 0 && capture == cudaStreamCaptureStatusNone;
  LoadPlan plan{};
  // TMA where a tile is whole boxes of whole pages: pages of whole tiles, or powers of two
  // from 16 keys (a bulk copy of scale bytes is at least 16), with 16-byte scale rows.
  const int bs = p.block_size;
  plan.box = bs % kN == 0 ? kN : bs;
  plan.tma = (bs % kN == 0 || (bs >= 16 && kN % bs == 0)) && al16(p.k_scale) && al16(p.v_scale) &&
             (p.ks_stride0 | p.ks_stride1 | p.vs_stride0 | p.vs_stride1) % 16 == 0;
  CUtensorMap kmap{}, vmap{};
  if (plan.tma &&
      (!encode_pool(&kmap, p, p.k_pool, p.k_stride0, p.k_stride1, p.k_stride2, plan.box) ||
       !encode_pool(&vmap, p, p.v_pool, p.v_stride0, p.v_stride1, p.v_stride2, plan.box)))
    plan.tma = 0;  // a layout the encoder refuses: gathered like any other page size
  // Requests of up to 16 rows and larger trees take kernels of their own; each skips the other's
  // requests, and the host leaves out a kernel that it knows to be without any.
  const int grid = std::min(sms, kMaxCtas);
  const int64_t least = static_cast<int64_t>(known ? std::max(p.min_nodes, 1) : 1) * p.groups;
  const int64_t most = known ? static_cast<int64_t>(p.max_nodes) * p.groups : kFewRows + 1;
  if (least <= kFewRows) {
    rc = most <= 8 ? launch_few<1, kWide, QT>(p, plan, kmap, vmap, grid, true, stream)
                   : launch_few<2, kWide, QT>(p, plan, kmap, vmap, grid, most <= kFewRows, stream);
    if (rc != JT_OK || most <= kFewRows) return rc;
  }
  const int64_t rows = static_cast<int64_t>(p.total_queries) * p.groups;
  CUtensorMap qmap{};
  if (!encode_queries(&qmap, carve(p.workspace, p.total_queries, p.groups, p.num_kv_heads).q_terms, rows,
                      p.num_kv_heads * Smem<kWide>::kTerms))
    return jt_fail(JT_ERR_CUDA, "tree_attn_fp8: cuTensorMapEncodeTiled rejected the query terms");
  rc = jt_cuda_check(cudaFuncSetAttribute(tree_attn_fp8_kernel<kWide>,
                                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                                              Smem<kWide>::kBytes),
                         "tree_attn_fp8 smem attribute");
  if (rc != JT_OK) return rc;
  const int64_t split = (rows * p.num_kv_heads + 15) / 16, mask = (p.total_queries + 7ll) / 8;
  if (split + mask > 0x7fffffff || rows > 0x7fffffff)
    return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: too many query rows");
  tree_attn_fp8_split_kernel<kWide, QT><<<static_cast<unsigned>(split + mask), 256, 0, stream>>>(
      p, static_cast<unsigned>(split));
  rc = jt_cuda_check(cudaGetLastError(), "tree_attn_fp8 query split launch");
  if (rc != JT_OK) return rc;
  rc = launch_dependent(tree_attn_fp8_kernel<kWide>, dim3(grid), kThreads, Smem<kWide>::kBytes, stream,
                        "tree_attn_fp8 launch", p, kmap, vmap, qmap, plan);
  if (rc != JT_OK) return rc;
  return launch_dependent(tree_attn_fp8_merge_kernel<kWide>, dim3(grid, 8 * Smem<kWide>::kTiles), kM,
                          0, stream, "tree_attn_fp8 merge launch", p, grid,
                           static_cast<int>(least > kFewRows ? kFewRows + 1 : 1));
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
  return workspace_bytes(total_queries, groups, num_kv_heads);
}

extern "C" int jt_tree_attn_fp8_launch(const JtTreeAttnFp8Params* p, cudaStream_t stream) {
  if (p == nullptr) return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: null params");
  if (p->num_requests < 1 || p->total_queries < 1 || p->num_kv_heads < 1 || p->groups < 1 ||
      p->groups > kM || p->block_size < 1 || p->num_blocks < 1 || p->num_blocks > 0x7fffffff ||
      p->table_width < 1)
    return jt_fail(JT_ERR_INVALID, "tree_attn_fp8: invalid geometry");
  if (p->head_dim < 16 || p->head_dim > kD || p->head_dim % 16 != 0)
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
  if (!al16(p->q) || !al16(p->out) || !al16(p->k_pool) || !al16(p->v_pool) ||
      (p->q_stride0 | p->q_stride1 | p->out_stride0 | p->out_stride1) % 8 != 0 ||
      (p->k_stride0 | p->k_stride1 | p->k_stride2 | p->v_stride0 | p->v_stride1 | p->v_stride2) % 16 != 0)
    return jt_fail(JT_ERR_INVALID,
                   "tree_attn_fp8: queries, output and pool rows must start on 16 bytes");
  const int64_t need = workspace_bytes(p->total_queries, p->groups, p->num_kv_heads);
  if (p->workspace == nullptr || p->workspace_bytes < need ||
      (reinterpret_cast<uintptr_t>(p->workspace) & 255u) != 0)
    return jt_fail(JT_ERR_WORKSPACE, "tree_attn_fp8: workspace of %lld bytes required (got %lld)",
                   static_cast<long long>(need), static_cast<long long>(p->workspace_bytes));
  int dev = 0, sms = 0;
  int rc = jt_cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
  if (rc != JT_OK) return rc;
  rc = jt_cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "SM count");
  if (rc != JT_OK) return rc;
  if (p->dtype == JT_F16) return launch<true, __half>(*p, sms, stream);
  return p->out_dtype == JT_BF16 ? launch<false, __nv_bfloat16>(*p, sms, stream)
                                 : launch<true, __nv_bfloat16>(*p, sms, stream);
}
